"""Workloads of the key-value cache in 8 bits (appending to it, attention over it), and of beam search over such caches: its selection, and the reordering of sequences.

`prepare` makes what a serving program has in hand before the call (projections of new tokens, tables of blocks and lengths, the cache with what earlier calls have
put there; logits and scores of beams), `run` makes the calls, in plain torch or through this package.

A row (the keys, or the values, of a token and head) is kept as eight-bit floating-point numbers of four significant bits (e4m3) and a power of two 2^k: k is the least for which
the largest of the row is at most 448 * 2^k, between bounds that the type of the inputs sets.  A cache is cut into blocks of T tokens: T is the largest power of two for which
T rows fit a page.  `table[b][i]` is the block that holds tokens i*T .. i*T+T-1 of sequence b; `lens[b]` counts its tokens, the new ones among them, and the new tokens of sequence
b are rows starts[b] .. starts[b+1]-1 of the packed inputs.  The token at position p sees position t if t <= p and, with a window, if p - t < window or t < sinks.  Query head h
reads the keys of head h // (heads / kv).
"""
import itertools
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
# powers of two of a row, and the largest number that is kept, by the type of the rows
_POWERS = {torch.bfloat16: (-110, 120), torch.float16: (-24, 8)}
_MOST = {torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 1.875 * 2.0 ** 15}


def listed():
    return [
        # one conversation, one new token, with norms of queries and keys: nothing but latency
        {"name": "append_one", "op": "append", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 513, "new": 1, "rotary": "half", "rot": 128, "norm": True},
        # a batch of prompts of all lengths going in
        {"name": "append_prompts", "op": "append", "batch": 8, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 4100, "new": 4099, "rotary": "half", "rot": 128, "norm": True},
        # one conversation shortly after its start: latency
        {"name": "token_short", "op": "attend", "batch": 1, "heads": 16, "kv": 4, "dim": 64, "page": 4096, "dtype": "f16",
         "len": 201, "new": 1, "window": 0, "sinks": 0},
        # as many conversations as a card serves at a time
        {"name": "token_largest", "op": "attend", "batch": 128, "heads": 64, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 8192, "new": 1, "window": 0, "sinks": 0},
        # one conversation over a whole library: the length is all the work there is to share out
        {"name": "token_long", "op": "attend", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 16384, "dtype": "bf16",
         "len": 262121, "new": 1, "window": 0, "sinks": 0},
        # a piece of a long prompt, the rest of it in the cache already
        {"name": "prompt_piece", "op": "attend", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 33000, "new": 500, "window": 0, "sinks": 0},
        # prompts of all lengths through a layer with a sliding window
        {"name": "prompts_window", "op": "attend", "batch": 4, "heads": 32, "kv": 4, "dim": 96, "page": 8192, "dtype": "f16",
         "len": 8000, "new": 8000, "window": 1024, "sinks": 4},
        # one request of four beams: latency
        {"name": "select_one", "op": "select", "batch": 1, "beams": 4, "width": 8, "vocab": 32000, "dtype": "bf16"},
        # a batch of requests, with room for beams that end
        {"name": "select_batch", "op": "select", "batch": 32, "beams": 4, "width": 8, "vocab": 128000, "dtype": "bf16"},
        # wide beams, logits as a 32-bit head leaves them, rows that end nowhere in particular
        {"name": "select_largest", "op": "select", "batch": 48, "beams": 16, "width": 32, "vocab": 150001, "dtype": "f32"},
        # one request of four beams behind a selection: latency
        {"name": "reorder_one", "op": "reorder", "batch": 1, "beams": 4, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16", "eight": True, "len": 525},
        # many requests, in 16 bits
        {"name": "reorder_batch", "op": "reorder", "batch": 64, "beams": 8, "kv": 8, "dim": 128, "page": 8192, "dtype": "bf16", "eight": False, "len": 1999},
    ]


def _spread(rng, low, high):
    """a whole number between low and high, spread over the logarithm"""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["append", "token", "token", "prompt", "prompt", "select", "select", "reorder"])
    if kind == "select":
        beams = _spread(rng, 1, 32)
        vocab = _spread(rng, 500, 160000)
        most = max(1, min(64, 110_000_000 // (beams * vocab)))
        return {"op": "select", "batch": _spread(rng, 1, most), "beams": beams, "width": rng.choice([beams, 2 * beams, rng.randint(1, 64)]), "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    page, dtype = rng.choice([4096, 4096, 8192, 16384]), rng.choice(["bf16", "bf16", "f16"])
    if kind == "reorder":
        beams = rng.randint(2, 16)
        batch = _spread(rng, 1, 64)
        return {"op": "reorder", "batch": batch, "beams": beams, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "eight": rng.random() < 0.6,
                "len": _spread(rng, 5, max(8, min(4000, 60_000_000 // (batch * beams * kv * dim))))}
    case = {"op": "append" if kind == "append" else "attend", "heads": kv * group, "kv": kv, "dim": dim, "page": page, "dtype": dtype}
    row = 2 * kv * dim                                       # bytes of a token's keys and values
    if kind == "append":
        if rng.random() < 0.5:
            batch, new = _spread(rng, 1, 200), 1
        else:
            batch = _spread(rng, 1, 12)
            new = _spread(rng, 2, 4096)
        case.update(batch=batch, new=new, len=new + rng.randint(0, 500))
        case.update(rotary=rng.choice(["half", "pairs"]), rot=rng.choice([dim, dim, dim // 32 * 16]), norm=rng.random() < 0.5)
        return case
    windowed = rng.random() < 0.35
    case.update(window=_spread(rng, 16, 4096) if windowed else 0, sinks=rng.choice([0, 1, 4, 64]) if windowed else 0)
    if kind == "token":
        batch = _spread(rng, 1, 160)
        case.update(batch=batch, new=rng.choice([1, 1, 1, 2, 3]), len=_spread(rng, 3, max(4, min(262144, (1 << 30) // (row * batch)))))
        return case
    batch = _spread(rng, 1, 8)
    new = _spread(rng, 17, max(32, 8192 // batch))
    case.update(batch=batch, new=new, len=new + rng.choice([0, 0, _spread(rng, 1, 16384 // batch)]))
    while work(case)["flops"] > 2.8e11:                      # many wide heads: not that many tokens
        case["len"] -= case["new"] - case["new"] // 2
        case["new"] //= 2
    return case


def _block_tokens(case):
    return 1 << ((case["page"] // (case["dim"] * (1 if case.get("eight", True) else 2))).bit_length() - 1)


def _lengths(case):
    """(tokens of each sequence, how many of them are new): the first has the case's lengths, the others as many or fewer"""
    rng = random.Random(17)
    news = [case["new"]] + [case["new"] if case["new"] <= 8 else rng.randint(max(1, case["new"] // 8), case["new"]) for _ in range(case["batch"] - 1)]
    before = case["len"] - case["new"]
    return [n + (before if i == 0 else rng.randint(before // 2, before)) for i, n in enumerate(news)], news


def _beam_lengths(case):
    """tokens of each request: all its beams have as many"""
    rng = random.Random(29)
    return [case["len"]] + [rng.randint(max(1, case["len"] // 2), case["len"]) for _ in range(case["batch"] - 1)]


def _visible(case, lens, news):
    """pairs of a new token and a position it sees, and positions that any of a sequence's new tokens sees"""
    w, s = case.get("window", 0), case.get("sinks", 0)
    pairs = touched = 0
    for n, m in zip(lens, news):
        first = n - m
        if not w:
            pairs += m * first + m * (m + 1) // 2
            touched += n
            continue
        for p in (range(first, n) if m <= 8 else []):
            low = max(0, p - w + 1)
            pairs += p + 1 - low + min(s, low)
        if m > 8:
            p = torch.arange(first, n, dtype=torch.int64)
            low = (p - w + 1).clamp(min=0)
            pairs += int((p + 1 - low + low.clamp(max=s)).sum())
        low = max(0, first - w + 1)
        touched += n - low + min(s, low)
    return pairs, touched


def work(case):
    if case["op"] == "select":
        # every logit once: its exponential, and its place among the best
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * _SIZES[case["dtype"]] + case["batch"] * (4 * case["beams"] + 12 * case["width"]), "flops": 4 * n}
    if case["op"] == "reorder":
        # the copied rows in and out; what is read back afterwards: in and out; the tables in and out
        t, row = _block_tokens(case), 2 * case["kv"] * (case["dim"] + 1 if case["eight"] else 2 * case["dim"])
        lens = _beam_lengths(case)
        copied = sum((n % t) * (case["beams"] - (case["beams"] + 1) // 2) for n in lens)
        back = sum((n % t) * case["beams"] for n in lens)
        tables = sum(-(-n // t) * case["beams"] for n in lens)
        return {"bytes": 2 * copied * row + back * (row + 4 * case["kv"] * case["dim"]) + 8 * tables + 24 * len(lens) * case["beams"], "flops": 0}
    lens, news = _lengths(case)
    n, hq, hk, d = sum(news), case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        # projections in, queries out, keys and values into the cache and out again; each row of the two tables once for a token
        elems = n * (hq + 2 * hk) * d + n * hq * d + 2 * n * hk * d
        return {"bytes": 2 * elems + 2 * 2 * n * hk * (d + 1) + 4 * n * case["rot"], "flops": n * (hq + hk) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}
    pairs, touched = _visible(case, lens, news)
    return {"bytes": 2 * 2 * n * hq * d + 2 * touched * hk * (d + 1), "flops": 4 * pairs * hq * d}


# ---- inputs ----

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, dtype, *shape):
    """in pieces: the 32-bit numbers behind a large cache are twice its size"""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    step = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], step):
        out[i:i + step] = torch.randn((min(step, shape[0] - i),) + tuple(shape[1:]), generator=gen, device="cuda")
    return out


def _i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _starts(news):
    return _i32(itertools.accumulate(news, initial=0))


def _blocks(seed, counts, spare):
    """tables of as many blocks as are asked for, in no order, and the blocks behind them"""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed), dtype=torch.int64).to(torch.int32)
    table = torch.zeros(len(counts), max(counts), dtype=torch.int32)
    at = 0
    for b, k in enumerate(counts):
        table[b, :k] = order[at:at + k]
        at += k
    return total, table.cuda(), order[at:].cuda()


def _old_rows(gen, dt, m, hk, d):
    """keys and values of the tokens that are in the cache beforehand: tokens of different sizes, values around something"""
    k, v = _randn(gen, dt, m, hk, d), _randn(gen, dt, m, hk, d)
    v += (0.5 * torch.randn(hk, d, generator=gen, device="cuda")).to(dt)
    v *= torch.exp(torch.rand(m, 1, 1, generator=gen, device="cuda") - 0.5).to(dt)
    return k, v


def _inputs(case, seed):
    """What the operator is given, apart from the cache itself, and the keys and values that are in the cache beforehand."""
    gen, dt = _generator(seed), _DTYPES[case["dtype"]]
    if case["op"] == "select":
        # a few tokens stand out in each row, and the beams of a request lie close together
        rows, v = case["batch"] * case["beams"], case["vocab"]
        logits = _randn(gen, dt, rows, v)
        step = max(1, (1 << 26) // v)
        for i in range(0, rows, step):
            part = logits[i:i + step]
            part *= 3
            at = torch.arange(40, device="cuda") * (v // 40) + torch.randint(0, v // 40, (part.shape[0], 40), generator=gen, device="cuda")
            part.scatter_(1, at, (12 * torch.rand(part.shape[0], 40, generator=gen, device="cuda")).to(dt))
        scores = -20 * torch.rand(case["batch"], 1, generator=gen, device="cuda") - 4 * torch.rand(case["batch"], case["beams"], generator=gen, device="cuda")
        return {"logits": logits, "scores": scores}
    hk, d, t = case["kv"], case["dim"], _block_tokens(case)
    if case["op"] == "reorder":
        # half of the beams are continued, some of them more than once
        per, beams = _beam_lengths(case), case["beams"]
        rng = random.Random(seed)
        parents = []
        for r in range(len(per)):
            kept = rng.sample(range(beams), (beams + 1) // 2)
            kept += [rng.choice(kept) for _ in range(beams - len(kept))]
            rng.shuffle(kept)
            parents += [r * beams + p for p in kept]
        lens = [n for n in per for _ in range(beams)]
        s = {"lens_list": lens, "block": t, "parents": _i32(parents), "lens": _i32(lens), "rests": [n % t for n in lens]}
        s["n_blocks"], s["table"], s["spare"] = _blocks(seed, [-(-n // t) for n in lens], len(lens))
        s["starts"] = _starts(s["rests"])
        s["old_k"], s["old_v"] = _old_rows(gen, dt, sum(lens), hk, d)
        s["before_list"] = lens
        return s
    hq = case["heads"]
    lens, news = _lengths(case)
    s = {"lens_list": lens, "news_list": news, "block": t}
    s["n_blocks"], s["table"], _ = _blocks(seed, [-(-n // t) for n in lens], 3)
    s["lens"], s["starts"] = _i32(lens), _starts(news)
    n = sum(news)
    if case["op"] == "append":
        # the output of one fused projection, its heads side by side; keys and queries of some heads are larger than of others
        qkv = _randn(gen, torch.float32, n, hq + 2 * hk, d)
        qkv *= torch.exp(torch.rand(hq + 2 * hk, 1, generator=gen, device="cuda") * 1.4)
        qkv = qkv.to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        s["q_norm"] = (1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dt) if case["norm"] else None
        s["k_norm"] = (1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dt) if case["norm"] else None
        angle = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        before = [a - b for a, b in zip(lens, news)]
    else:
        q = _randn(gen, torch.float32, n, hq, d)
        q *= torch.exp(torch.rand(hq, 1, generator=gen, device="cuda") * 1.4)          # some heads look at few tokens, some at many
        s["q"] = q.to(dt)
        before = lens
    # the tokens the cache holds beforehand, packed one sequence after the other
    s["before_list"] = before
    s["old_k"], s["old_v"] = _old_rows(gen, dt, sum(before), hk, d)
    return s


_serial = itertools.count()
_shared = {}


def _controller():
    """The store that all caches of this program lie on, and its controller.  Everything is resident in the cases here, so nothing is written back and the
    store needs no memory of its own."""
    import bam_amd
    if "ctrl" not in _shared:
        path = "/dev/libnvm-kv8-%d" % next(_serial)
        _shared["target"] = bam_amd.Target(path, 1 << 40, 512, backing=False, seed=7, n_io_threads=4)
        _shared["ctrl"] = bam_amd.Controller(path, 1, 0, queue_depth=256, n_queues=32)
    return _shared["ctrl"]


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "select":
        return s
    eight = case.get("eight", True)
    hk, d, t, dt = case["kv"], case["dim"], s["block"], _DTYPES[case["dtype"]]
    old_k, old_v, before = s.pop("old_k"), s.pop("old_v"), s["before_list"]
    s["one_each"] = case.get("new") == 1
    if own:
        import bam_amd
        s["cache"] = bam_amd.make_kv_cache(_controller(), s["n_blocks"], hk, d, page_size=case["page"], dtype=dt, stored=torch.float8_e4m3fn if eight else None)
        assert s["cache"].block_tokens == t
        if old_k.shape[0]:
            s["cache"].append(old_k, old_v, _i32(before), s["table"], starts=_starts(before))
        # the pages that the call writes to are in the cache too, as for a program that has used these blocks before; what they hold is not what the call puts there
        if case["op"] == "append":
            s["cache"].append(s["v"], s["k"], s["lens"], s["table"], starts=s["starts"])
        if case["op"] == "reorder":
            n = s["spare"].numel()
            rows = old_k[:1].expand(n * t, -1, -1)
            s["cache"].append(rows, rows, _i32([t] * n), s["spare"][:, None], starts=_starts([t] * n))
        torch.cuda.synchronize()
        return s
    kind = torch.uint8 if eight else dt
    s["k_pool"] = torch.zeros(s["n_blocks"], hk, t, d, dtype=kind, device="cuda")
    s["v_pool"] = torch.zeros_like(s["k_pool"])
    if eight:
        s["k_power"] = torch.ones(s["n_blocks"], hk, t, dtype=torch.float32, device="cuda")
        s["v_power"] = torch.ones_like(s["k_power"])
    at = 0
    for b, n in enumerate(before):
        for i in range(0, n, 16384):
            pos = torch.arange(i, min(n, i + 16384), device="cuda")
            block, inside = s["table"][b].long()[pos // t], pos % t
            _plain_put(s, "k", block, inside, old_k[at + i:at + i + pos.numel()])
            _plain_put(s, "v", block, inside, old_v[at + i:at + i + pos.numel()])
        at += n
    if case["op"] == "append":
        # positions and blocks of the new tokens are found within the call
        s["row_of"] = torch.arange(sum(s["news_list"]), device="cuda")
    return s


# ---- the operators in plain torch ----

def _plain_eight(x, dt):
    """numbers in 32 bits as e4m3 (their bytes), and the power of two of each row"""
    low, high = _POWERS[dt]
    x = x.float().clamp(-_MOST[dt], _MOST[dt])
    part, power = torch.frexp(x.abs().amax(dim=-1, keepdim=True))
    power = (power - 9 + (part > 0.875).int()).clamp(low, high)
    by = ((power + 127) << 23).view(torch.float32)                     # 2^power, from its exponent
    return (x / by).to(torch.float8_e4m3fn).view(torch.uint8), by[..., 0]


def _plain_put(s, what, block, inside, x):
    if "k_power" in s:
        x, by = _plain_eight(x, _DTYPES[s["case"]["dtype"]])
        s[what + "_power"][block, :, inside] = by
    s[what + "_pool"][block, :, inside] = x


def _plain_get(s, what, *at):
    x = s[what + "_pool"][at]
    if "k_power" not in s:
        return x.float()
    return x.view(torch.float8_e4m3fn).float() * s[what + "_power"][at][..., None]


def _plain_rotated(x, weight, cos, sin, rot, style):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS) * weight.float()
    turned, rest = x[..., :rot], x[..., rot:]
    c, s = cos[:, None, :], sin[:, None, :]
    if style == "half":
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1)


def _plain_append(s):
    case, t = s["case"], s["block"]
    dt = s["q"].dtype
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, s["row_of"], right=True) - 1
    pos = s["lens"].long()[seq] - starts[seq + 1] + s["row_of"]
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _plain_rotated(s["q"], s["q_norm"], cos, sin, case["rot"], case["rotary"]).to(dt)
    block, inside = s["table"].long()[seq, pos // t], pos % t
    _plain_put(s, "k", block, inside, _plain_rotated(s["k"], s["k_norm"], cos, sin, case["rot"], case["rotary"]))
    _plain_put(s, "v", block, inside, s["v"])
    heads = slice(None)
    return q, _plain_get(s, "k", block, heads, inside).to(dt), _plain_get(s, "v", block, heads, inside).to(dt)


def _plain_attend(s):
    case = s["case"]
    hq, hk, d, w, sinks, t = case["heads"], case["kv"], case["dim"], case["window"], case["sinks"], s["block"]
    out = torch.empty_like(s["q"])
    row = 0
    for b, (n, m) in enumerate(zip(s["lens_list"], s["news_list"])):
        blocks = s["table"][b, :-(-n // t)].long()
        q = s["q"][row:row + m].float().view(m, hk, hq // hk, d).permute(1, 0, 2, 3).reshape(hk, -1, d)           # [hk, m * group, d]
        pos = torch.arange(n - m, n, device="cuda").repeat_interleave(hq // hk)
        k = _plain_get(s, "k", blocks).permute(1, 3, 0, 2).reshape(hk, d, -1)[:, :, :n].contiguous()              # [hk, d, n]
        v = _plain_get(s, "v", blocks).transpose(0, 1).reshape(hk, -1, d)[:, :n].contiguous()                     # [hk, n, d]
        keys = torch.arange(n, device="cuda")
        got = torch.empty_like(q)
        step = max(1, (1 << 28) // (hk * n))
        for i in range(0, q.shape[1], step):
            p = pos[i:i + step, None]
            seen = keys[None] <= p
            if w:
                seen &= (p - keys[None] < w) | (keys[None] < sinks)
            score = torch.matmul(q[:, i:i + step], k) * d ** -0.5
            score.masked_fill_(~seen, float("-inf"))
            score -= score.amax(dim=-1, keepdim=True)
            score.exp_()
            got[:, i:i + step] = torch.matmul(score, v) / score.sum(dim=-1, keepdim=True)
        out[row:row + m] = got.view(hk, m, hq // hk, d).permute(1, 0, 2, 3).reshape(m, hq, d)
        row += m
    return out


def _plain_select(s):
    """in 64 bits: sums of different beams lie next to each other"""
    case = s["case"]
    b, n, v, width = case["batch"], case["beams"], case["vocab"], case["width"]
    x = s["logits"].double()
    top = x.amax(dim=1, keepdim=True)
    offset = s["scores"].double().view(-1, 1) - top - torch.log((x - top).exp_().sum(dim=1, keepdim=True))
    x += offset
    # the best of each beam, in order, and those of all beams; equal ones by their place
    best, at = _plain_best(x, min(width, v))
    at += torch.arange(n, device="cuda").repeat(b)[:, None] * v
    best, order = _plain_best(best.view(b, -1), width)
    at = at.view(b, -1).gather(1, order)
    return best.float(), (torch.arange(b, device="cuda")[:, None] * n + at // v).int(), (at % v).int()


def _plain_best(x, k):
    """the k largest of each row and where they are, equal ones in the order of their places"""
    least = torch.topk(x, k, dim=1).values[:, -1:]
    # those above the k-th largest, and the first of those equal to it
    above = x > least
    equal = x == least
    room = k - above.sum(dim=1, keepdim=True)
    taken = above | (equal & (equal.cumsum(dim=1) <= room))
    at = taken.nonzero()[:, 1].view(-1, k)
    values, order = torch.sort(x.gather(1, at), dim=1, descending=True, stable=True)
    return values, at.gather(1, order)


def _plain_reorder(s):
    t = s["block"]
    parents, n = s["parents"].long(), s["parents"].numel()
    lens = s["lens"][parents]
    same = parents[:, None] == parents[None]
    partly = lens % t != 0
    copies = same.tril(-1).any(dim=1) & partly                          # all but the first child of each
    last = (lens.long() // t).clamp(max=s["table"].shape[1] - 1)
    table = s["table"][parents]
    table = table.masked_fill(torch.arange(table.shape[1], device="cuda") * t >= lens[:, None], -1)
    at = torch.arange(n, device="cuda")
    source = s["table"][parents, last]
    target = torch.where(copies, s["spare"], source)
    table[at, last] = torch.where(copies, s["spare"], table[at, last])
    for what in ("k", "v"):
        s[what + "_pool"][target.long()] = s[what + "_pool"][source.long()]
        if "k_power" in s:
            s[what + "_power"][target.long()] = s[what + "_power"][source.long()]
    # the last blocks of those that nobody continues, in order, in place of the spare ones that were used
    old = torch.arange(s["lens"].numel(), device="cuda")
    free = ~(parents[None] == old[:, None]).any(dim=1) & (s["lens"] % t != 0)
    freed = s["table"][old, (s["lens"].long() // t).clamp(max=s["table"].shape[1] - 1)][torch.argsort((~free).int(), stable=True)]
    rank = copies.int().cumsum(0) - 1
    again = torch.where(rank < free.sum(), freed[rank.clamp(0, old.numel() - 1)], torch.full_like(s["spare"], -1))
    spare = torch.where(copies, again, s["spare"])
    # the rows of the last blocks
    row = torch.arange(sum(s["rests"]), device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    inside = row - starts[seq]
    block = table[seq, last[seq]].long()
    heads, dt = slice(None), _DTYPES[s["case"]["dtype"]]
    return lens, table, spare, _plain_get(s, "k", block, heads, inside).to(dt), _plain_get(s, "v", block, heads, inside).to(dt)


def run(s):
    case = s["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}[case["op"]](s)
    if case["op"] == "select":
        import bam_amd
        return bam_amd.beam_select(s["logits"], s["scores"], width=case["width"])
    if case["op"] == "reorder":
        lens, table, spare = s["cache"].reorder(s["parents"], s["lens"], s["table"], s["spare"])
        k, v = s["cache"].read(sum(s["rests"]), lens, table, starts=s["starts"])
        return lens, table, spare, k, v
    starts = None if s["one_each"] else s["starts"]
    if case["op"] == "append":
        q = s["cache"].append(s["k"], s["v"], s["lens"], s["table"], starts=starts, q=s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=_EPS,
                              cos=s["cos"], sin=s["sin"], rotary=case["rotary"])
        k, v = s["cache"].read(s["q"].shape[0], s["lens"], s["table"], starts=starts)
        return q, k, v
    return s["cache"].attend(s["q"], s["lens"], s["table"], starts=starts, max_new=case["new"], window=case["window"], sinks=case["sinks"])


# ---- the definition, in 64 bits ----

def _exact_eight(x, dt):
    """what rows are kept as, without the eight-bit type: multiples of an eighth of the largest power of two in each number (powers of two by way of their exponents: exact)"""
    low, high = _POWERS[dt]

    def two_to(n):
        return ((n.long() + 1023) << 52).view(torch.float64)

    x = x.double().clamp(-_MOST[dt], _MOST[dt])
    top = x.abs().amax(-1, keepdim=True)
    power = torch.full_like(top, high)
    for k in range(high - 1, low - 1, -1):
        power = torch.where(top <= 448 * 2.0 ** k, torch.full_like(top, k), power)
    y = x / two_to(power)
    unit = two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.round(y / unit) * unit * two_to(power)


def _exact_head_rows(x, weight, pos, rot, style, cos, sin):
    """rows [n, d] of one head: each plane of the rotation as a complex number"""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / x.shape[1] + _EPS) * weight.double()
    turn = torch.complex(cos.double()[pos], sin.double()[pos])
    i = torch.arange(rot // 2, device=x.device)
    re, im = (i, i + rot // 2) if style == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(x[:, re], x[:, im]) * turn
    y = x.clone()
    y[:, re], y[:, im] = z.real, z.imag
    return y


def _exact_select(case, s):
    """beam by beam; which they are is not a computed number"""
    best = []
    for b in range(case["batch"]):
        sums = []
        for i in range(case["beams"]):
            row = s["logits"][b * case["beams"] + i].double()
            sums.append(torch.sort(row, descending=True).values[:case["width"]] - torch.logsumexp(row, 0) + s["scores"][b, i].double())
        best.append(torch.sort(torch.cat(sums), descending=True).values[:case["width"]])
    return torch.stack(best), None, None


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "select":
        return _exact_select(case, s)
    hk, d, dt = case["kv"], case["dim"], _DTYPES[case["dtype"]]
    if case["op"] == "reorder":
        first = list(itertools.accumulate(s["lens_list"], initial=0))
        rows = [range(first[p] + n - r, first[p] + n) for p, n, r in zip(s["parents"].tolist(), s["lens_list"], s["rests"])]
        at = torch.tensor(list(itertools.chain.from_iterable(rows)), dtype=torch.int64, device="cuda")
        k, v = (_exact_eight(x[at], dt) if case["eight"] else x[at].double() for x in (s["old_k"], s["old_v"]))
        return None, None, None, k, v
    hq = case["heads"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(s["lens_list"], s["news_list"])]).cuda()
        q = torch.stack([_exact_head_rows(s["q"][:, h], s["q_norm"], pos, case["rot"], case["rotary"], s["cos"], s["sin"]) for h in range(hq)], 1)
        k = torch.stack([_exact_eight(_exact_head_rows(s["k"][:, h], s["k_norm"], pos, case["rot"], case["rotary"], s["cos"], s["sin"]), dt) for h in range(hk)], 1)
        return q, k, _exact_eight(s["v"], dt)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = row = 0
    for n, m in zip(s["lens_list"], s["news_list"]):
        t = torch.arange(n, dtype=torch.int64, device="cuda")
        rows = max(1, (1 << 26) // n)
        for g in range(hk):
            k, v = _exact_eight(s["old_k"][at:at + n, g], dt), _exact_eight(s["old_v"][at:at + n, g], dt)
            for h in range(g * (hq // hk), (g + 1) * (hq // hk)):
                for i in range(0, m, rows):
                    p = torch.arange(n - m + i, n - m + min(m, i + rows), dtype=torch.int64, device="cuda")[:, None]
                    hidden = t[None] > p
                    if case["window"]:
                        hidden |= (t[None] <= p - case["window"]) & (t[None] >= case["sinks"])
                    logit = s["q"][row + i:row + i + p.shape[0], h].double() @ k.T / math.sqrt(d)
                    logit[hidden] = -math.inf
                    out[row + i:row + i + p.shape[0], h] = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True)) @ v
        at += n
        row += m
    return out
