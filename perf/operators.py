"""Workloads of the key-value cache that is kept in the pages of an array: appending to it, and attention over it.

`prepare` makes what a serving program has in hand before the call (the projections of the new tokens, the tables of blocks and
lengths, the cache with what earlier calls have put there), `run` makes the calls, in plain torch or through this package.

A cache is cut into blocks of T tokens: T is the largest power of two for which T rows of one head fit a page.  `table[b][i]` is the block that holds tokens
i*T .. i*T+T-1 of sequence b; `lens[b]` counts its tokens, the new ones among them, and the new tokens of sequence b are rows
starts[b] .. starts[b+1]-1 of the packed inputs.  The token at position p sees position t if t <= p and, with a window, if p - t < window or
t < sinks.  Query head h reads the keys of head h // (heads / kv).
"""
import itertools
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-6


def listed():
    return [
        # one conversation, one new token, with norms of queries and keys: nothing but latency
        {"name": "append_one", "op": "append", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 513, "new": 1, "rotary": "half", "rot": 128, "norm": True},
        # a decoding batch of which half of every head is rotated, in neighbouring pairs
        {"name": "append_batch", "op": "append", "batch": 64, "heads": 32, "kv": 4, "dim": 80, "page": 4096, "dtype": "f16",
         "len": 777, "new": 1, "rotary": "pairs", "rot": 32, "norm": False},
        # a batch of prompts of all lengths going in
        {"name": "append_prompts", "op": "append", "batch": 8, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 4100, "new": 4099, "rotary": "half", "rot": 128, "norm": True},
        # one conversation shortly after its start: latency
        {"name": "token_short", "op": "attend", "batch": 1, "heads": 16, "kv": 4, "dim": 64, "page": 4096, "dtype": "f16",
         "len": 201, "new": 1, "window": 0, "sinks": 0},
        # a decoding batch, contexts of all lengths
        {"name": "token_batch", "op": "attend", "batch": 64, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 4099, "new": 1, "window": 0, "sinks": 0},
        # one conversation over a whole library: the length is all the work there is to share out
        {"name": "token_long", "op": "attend", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 16384, "dtype": "bf16",
         "len": 262121, "new": 1, "window": 0, "sinks": 0},
        # four drafted tokens at a time, each head with keys of its own, a sliding window and four first tokens
        {"name": "drafts_window", "op": "attend", "batch": 24, "heads": 16, "kv": 16, "dim": 96, "page": 4096, "dtype": "f16",
         "len": 9001, "new": 4, "window": 2048, "sinks": 4},
        # as many conversations as a card serves at a time
        {"name": "token_largest", "op": "attend", "batch": 128, "heads": 64, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 8192, "new": 1, "window": 0, "sinks": 0},
        # a short question, all of it new
        {"name": "prompt_short", "op": "attend", "batch": 1, "heads": 16, "kv": 4, "dim": 64, "page": 4096, "dtype": "bf16",
         "len": 77, "new": 77, "window": 0, "sinks": 0},
        # a piece of a long prompt, the rest of it in the cache already
        {"name": "prompt_piece", "op": "attend", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 33000, "new": 500, "window": 0, "sinks": 0},
        # prompts of all lengths through a layer with a sliding window
        {"name": "prompts_window", "op": "attend", "batch": 4, "heads": 32, "kv": 4, "dim": 128, "page": 8192, "dtype": "f16",
         "len": 8000, "new": 8000, "window": 1024, "sinks": 4},
        # a whole document
        {"name": "prompt_largest", "op": "attend", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "page": 4096, "dtype": "bf16",
         "len": 16384, "new": 16384, "window": 0, "sinks": 0},
    ]


def _spread(rng, low, high):
    """a whole number between low and high, spread over the logarithm"""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["append", "token", "token", "prompt", "prompt"])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    case = {"op": "append" if kind == "append" else "attend", "heads": kv * group, "kv": kv, "dim": dim,
            "page": rng.choice([4096, 4096, 8192, 16384]), "dtype": rng.choice(["bf16", "bf16", "f16"])}
    row = 4 * kv * dim                                       # bytes of a token's keys and values
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
        case.update(batch=batch, new=rng.choice([1, 1, 1, 2, 3]), len=_spread(rng, 3, max(4, min(262144, (2 << 30) // (row * batch)))))
        return case
    batch = _spread(rng, 1, 8)
    new = _spread(rng, 17, max(32, 8192 // batch))
    case.update(batch=batch, new=new, len=new + rng.choice([0, 0, _spread(rng, 1, 16384 // batch)]))
    while work(case)["flops"] > 2e12:                        # many wide heads: not that many tokens
        case["len"] -= case["new"] - case["new"] // 2
        case["new"] //= 2
    return case


def _block_tokens(case):
    return 1 << ((case["page"] // (2 * case["dim"])).bit_length() - 1)


def _lengths(case):
    """(tokens of each sequence, how many of them are new): the first has the case's lengths, the others as many or fewer"""
    rng = random.Random(17)
    news = [case["new"]] + [case["new"] if case["new"] <= 8 else rng.randint(max(1, case["new"] // 8), case["new"]) for _ in range(case["batch"] - 1)]
    before = case["len"] - case["new"]
    return [n + (before if i == 0 else rng.randint(before // 2, before)) for i, n in enumerate(news)], news


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
    lens, news = _lengths(case)
    n, hq, hk, d = sum(news), case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        # projections in, queries out, keys and values into the cache and out again; each row of the two tables once for a token
        elems = n * (hq + 2 * hk) * d + n * hq * d + 2 * n * hk * d + 4 * n * hk * d
        return {"bytes": 2 * elems + 4 * n * case["rot"], "flops": n * (hq + hk) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}
    pairs, touched = _visible(case, lens, news)
    return {"bytes": 2 * (2 * n * hq * d + 2 * touched * hk * d), "flops": 4 * pairs * hq * d}


# ---- inputs ----

def _randn(gen, dtype, *shape):
    """in pieces: the 32-bit numbers behind a large cache are twice its size"""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    step = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], step):
        out[i:i + step] = torch.randn((min(step, shape[0] - i),) + tuple(shape[1:]), generator=gen, device="cuda")
    return out


def _inputs(case, seed):
    """What the operator is given, apart from the cache itself, and the keys and values that are in the cache beforehand."""
    dt, hq, hk, d, t = _DTYPES[case["dtype"]], case["heads"], case["kv"], case["dim"], _block_tokens(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lens, news = _lengths(case)
    s = {"lens_list": lens, "news_list": news, "block": t}
    blocks = [-(-n // t) for n in lens]
    s["n_blocks"] = sum(blocks) + 3
    order = torch.randperm(s["n_blocks"], generator=torch.Generator().manual_seed(seed), dtype=torch.int64).to(torch.int32)
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
    at = 0
    for b, k in enumerate(blocks):
        table[b, :k] = order[at:at + k]
        at += k
    s["table"] = table.cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = list(itertools.accumulate(news, initial=0))
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    n = starts[-1]
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
    m = sum(before)
    s["before_list"] = before
    s["old_k"] = _randn(gen, dt, m, hk, d)
    s["old_v"] = _randn(gen, dt, m, hk, d)
    s["old_v"] += (0.5 * torch.randn(hk, d, generator=gen, device="cuda")).to(dt)
    return s


_serial = itertools.count()
_shared = {}


def _controller():
    """The store that all caches of this program lie on, and its controller.  Everything is resident in the cases here, so nothing is written back and the
    store needs no memory of its own."""
    import bam_amd
    if "ctrl" not in _shared:
        path = "/dev/libnvm-kv%d" % next(_serial)
        _shared["target"] = bam_amd.Target(path, 1 << 40, 512, backing=False, seed=7, n_io_threads=4)
        _shared["ctrl"] = bam_amd.Controller(path, 1, 0, queue_depth=256, n_queues=32)
    return _shared["ctrl"]


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["one_each"] = case["new"] == 1
    hk, d, t = case["kv"], case["dim"], s["block"]
    old_k, old_v, before = s.pop("old_k"), s.pop("old_v"), s["before_list"]
    if own:
        import bam_amd
        s["cache"] = bam_amd.make_kv_cache(_controller(), s["n_blocks"], hk, d, page_size=case["page"], dtype=_DTYPES[case["dtype"]])
        assert s["cache"].block_tokens == t
        if old_k.shape[0]:
            have = torch.tensor(before, dtype=torch.int32, device="cuda")
            old_starts = torch.tensor(list(itertools.accumulate(before, initial=0)), dtype=torch.int32, device="cuda")
            s["cache"].append(old_k, old_v, have, s["table"], starts=old_starts)
        if case["op"] == "append":
            # the pages of the new tokens are in the cache too, as for a program that has used these blocks before
            s["cache"].append(s["k"], s["v"], s["lens"], s["table"], starts=s["starts"])
        torch.cuda.synchronize()
        return s
    s["k_pool"] = torch.zeros(s["n_blocks"], hk, t, d, dtype=old_k.dtype, device="cuda")
    s["v_pool"] = torch.zeros_like(s["k_pool"])
    at = 0
    for b, n in enumerate(before):
        pos = torch.arange(n, device="cuda")
        block = s["table"][b].long()[pos // t]
        s["k_pool"][block, :, pos % t] = old_k[at:at + n]
        s["v_pool"][block, :, pos % t] = old_v[at:at + n]
        at += n
    if case["op"] == "append":
        # positions and blocks of the new tokens are found within the call
        s["row_of"] = torch.arange(sum(s["news_list"]), device="cuda")
    return s


# ---- the operators in plain torch ----

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
    k = _plain_rotated(s["k"], s["k_norm"], cos, sin, case["rot"], case["rotary"]).to(dt)
    block, inside = s["table"].long()[seq, pos // t], pos % t
    s["k_pool"][block, :, inside] = k
    s["v_pool"][block, :, inside] = s["v"]
    return q, s["k_pool"][block, :, inside], s["v_pool"][block, :, inside]


def _plain_attend(s):
    case, t = s["case"], s["block"]
    hq, hk, d, w, sinks = case["heads"], case["kv"], case["dim"], case["window"], case["sinks"]
    out = torch.empty_like(s["q"])
    row = 0
    for b, (n, m) in enumerate(zip(s["lens_list"], s["news_list"])):
        blocks = s["table"][b, :-(-n // t)].long()
        q = s["q"][row:row + m].float().view(m, hk, hq // hk, d).permute(1, 0, 2, 3).reshape(hk, -1, d)           # [hk, m * group, d]
        pos = torch.arange(n - m, n, device="cuda").repeat_interleave(hq // hk)
        k = s["k_pool"][blocks].permute(1, 3, 0, 2).reshape(hk, d, -1)[:, :, :n].float().contiguous()             # [hk, d, n]
        v = s["v_pool"][blocks].transpose(0, 1).reshape(hk, -1, d)[:, :n].float().contiguous()                    # [hk, n, d]
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


def run(s):
    case = s["case"]
    if not own:
        return _plain_append(s) if case["op"] == "append" else _plain_attend(s)
    starts = None if s["one_each"] else s["starts"]
    if case["op"] == "append":
        q = s["cache"].append(s["k"], s["v"], s["lens"], s["table"], starts=starts, q=s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=_EPS,
                              cos=s["cos"], sin=s["sin"], rotary=case["rotary"])
        k, v = s["cache"].read(s["q"].shape[0], s["lens"], s["table"], starts=starts)
        return q, k, v
    return s["cache"].attend(s["q"], s["lens"], s["table"], starts=starts, max_new=case["new"], window=case["window"], sinks=case["sinks"])


# ---- the definition, in 64 bits ----

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


def exact(case, seed):
    s = _inputs(case, seed)
    hq, hk, d = case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(s["lens_list"], s["news_list"])]).cuda()
        q = torch.stack([_exact_head_rows(s["q"][:, h], s["q_norm"], pos, case["rot"], case["rotary"], s["cos"], s["sin"]) for h in range(hq)], 1)
        k = torch.stack([_exact_head_rows(s["k"][:, h], s["k_norm"], pos, case["rot"], case["rotary"], s["cos"], s["sin"]) for h in range(hk)], 1)
        return q, k, s["v"].double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = row = 0
    for n, m in zip(s["lens_list"], s["news_list"]):
        t = torch.arange(n, dtype=torch.int64, device="cuda")
        rows = max(1, (1 << 26) // n)
        for g in range(hk):
            k, v = s["old_k"][at:at + n, g].double(), s["old_v"][at:at + n, g].double()
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
