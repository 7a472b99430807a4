"""The calls that the key-value cache operators' speed is measured on.

Four operators share one cache of 8-bit codes: `append` writes new tokens into
it, `attention` reads all of a sequence, `select` chooses the blocks of tokens
worth reading, `sparse` reads those. `run` computes them in plain torch
operations in 32 bits, or with the framework's kernels where `own` is set.

The cache: `blocks` of `block` tokens; for each block and kv head the codes of
its keys (tokens x dim) and values (dim x tokens), a scale for each of the two,
and the largest and least key code for each dimension. `table` gives the block
of each part of a sequence, `lengths` the sequences' tokens, those of the
current call included (the last ones).
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEAST = -100  # exponent of the least scale


def _case(name, op, dtype, seqs, heads, kv_heads, dim, block, least, most, new=1, ragged=False, idle=0, lse=False,
          count=0, sink=0, recent=0):
    c = {"op": op, "dtype": dtype, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
         "least": least, "most": most, "new": new, "ragged": ragged, "idle": idle, "lse": lse, "count": count,
         "sink": sink, "recent": recent}
    return {"name": name, **c} if name else c


def listed():
    return [
        # every step of a serving loop writes one token per sequence
        _case("append_step", "append", "bf16", 64, 32, 8, 128, 64, 500, 9000),
        # prompts of different lengths enter the cache, some of them behind an earlier part
        _case("append_prompts", "append", "f16", 16, 32, 8, 128, 64, 40, 5000, new=4000, ragged=True),
        # one user, short conversation: the launch and the latency of a single step
        _case("step_one", "attention", "bf16", 1, 32, 8, 128, 64, 700, 700),
        # a serving batch in mid-flight, two of its slots idle
        _case("step_batch", "attention", "bf16", 64, 32, 8, 128, 64, 500, 12000, idle=2),
        # two long documents; the sums are kept to be joined with another part of the context
        _case("step_long", "attention", "f16", 2, 16, 2, 128, 64, 400001, 600000, lse=True),
        # a draft's five tokens verified at once, an odd group of heads, narrow rows, small blocks
        _case("verify_draft", "attention", "bf16", 24, 21, 3, 64, 16, 200, 3500, new=5, ragged=True),
        # prompts that enter in chunks over what is cached already
        _case("chunk", "attention", "bf16", 2, 32, 8, 128, 64, 6000, 10000, new=2048),
        # short prompts of odd lengths, one head per kv head, 96 dimensions
        _case("prompts_odd", "attention", "f16", 7, 12, 12, 96, 32, 1, 1500, new=1300, ragged=True),
        # the blocks for one step of a batch with long contexts
        _case("select_step", "select", "bf16", 16, 32, 8, 128, 64, 60000, 131072, count=64, sink=1, recent=2),
        # the blocks for every token of a chunk
        _case("select_chunk", "select", "f16", 2, 32, 8, 128, 32, 20000, 40000, new=513, count=48, sink=1, recent=2),
        # that step's attention
        _case("sparse_step", "sparse", "bf16", 16, 32, 8, 128, 64, 60000, 131072, count=64, sink=1, recent=2),
        # that chunk's attention
        _case("sparse_chunk", "sparse", "f16", 2, 32, 8, 128, 32, 20000, 40000, new=513, count=48, sink=1, recent=2),
    ]


def _log(rng, a, b):
    return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most = {k: max(most.get(k, 0), w[k]) for k in w}
    while True:
        op = rng.choice(["append", "attention", "attention", "attention", "select", "sparse"])
        kv = rng.choice([1, 2, 3, 4, 5, 8, 8, 12, 16])
        group = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 12, 16])
        dim = rng.choice([64, 96, 128, 128, 192, 256])
        block = rng.choice([16, 32, 64, 64, 128])
        chunk = rng.random() < 0.4
        seqs = _log(rng, 1, 8 if chunk else 128)
        longest = _log(rng, 8, 4000 if op == "append" else 20000 if chunk else 200000)
        least = _log(rng, max(1, longest // 16), longest)
        new = _log(rng, 1, 2048) if chunk else rng.choice([1, 1, 1, 1, 2, 3, 5, 8])
        if op == "sparse":
            new = min(new, 256)
        idle = rng.choice([0, 0, 0, 1]) if seqs > 1 else 0
        count = _log(rng, 1, 128) if op in ("select", "sparse") else 0
        c = _case(None, op, rng.choice(["bf16", "f16"]), seqs, kv * group, kv, dim, block, least, longest, new=new,
                  ragged=new > 1 and rng.random() < 0.6, idle=idle, lse=op == "attention" and rng.random() < 0.3,
                  count=count, sink=min(count, rng.choice([0, 1, 2])) if count else 0,
                  recent=min(count, rng.choice([0, 1, 2])) if count else 0)
        w = work(c)
        lens, news = _lengths(c)
        blocks = [-(-n // block) for n in lens]
        logits = c["heads"] * seqs * max(news) * max(blocks) * block  # what the plain form holds at once
        stored = kv * dim * block * seqs * max(blocks)
        listwise = sum(news) * kv * count * block * dim
        if (w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and w["bytes"] > 2000 and stored < 1 << 31
                and (op != "attention" or logits < 1 << 31) and (op != "sparse" or listwise < 1 << 31)
                and (op != "select" or c["heads"] * sum(news) * max(blocks) < 1 << 29)
                # a selection leaves something out, and is not the forced blocks alone
                and (op != "select" or (max(blocks) >= 3 * count and count > c["sink"] + c["recent"]))):
            return c


def _lengths(c):
    """Tokens of each sequence, and how many of them are this call's: from the case alone."""
    r = random.Random("%s %s" % (c["seqs"], sorted((k, v) for k, v in c.items() if k not in ("name", "op"))))
    lens = [_log(r, c["least"], c["most"]) for _ in range(c["seqs"])]
    news = [_log(r, 1, c["new"]) if c["ragged"] else c["new"] for _ in lens]
    if c["op"] == "append" and c["new"] > 1:  # a prompt comes whole, or after an earlier part
        lens = [n if r.random() < 0.5 else n + r.randrange(200) for n in news]
    lens = [max(n, m) for n, m in zip(lens, news)]
    for b in range(c["idle"]):  # slots of the batch that hold no sequence: a query each, nothing to read
        lens[b], news[b] = 0, 1
    return lens, news


def _visible(c):
    """(tokens, blocks) that each query sees, as lists over the queries."""
    lens, news = _lengths(c)
    seen = [max(0, n - m + i + 1) for n, m in zip(lens, news) for i in range(m)]
    return seen, [-(-t // c["block"]) for t in seen]


def work(case):
    c = case
    lens, news = _lengths(c)
    heads, kv, dim, bs, t = c["heads"], c["kv_heads"], c["dim"], c["block"], sum(news)
    seen, seen_blocks = _visible(c)
    blocks = [-(-n // bs) for n in lens]
    if c["op"] == "append":
        t = sum(min(n, m) for n, m in zip(lens, news))
        touched = sum(-(-n // bs) - (n - m) // bs for n, m in zip(lens, news) if n >= m)
        return {"bytes": t * kv * dim * 6 + touched * kv * (2 * dim + 8), "flops": 0}
    rows = t * heads * dim * 2
    if c["op"] == "attention":
        return {"bytes": sum(lens) * kv * dim * 2 + sum(blocks) * kv * 8 + 2 * rows + (t * heads * 4 if c["lse"] else 0),
                "flops": 4 * heads * dim * sum(seen)}
    if c["op"] == "select":
        return {"bytes": sum(blocks) * kv * (2 * dim + 4) + rows + t * kv * c["count"] * 4,
                "flops": 4 * heads * dim * sum(seen_blocks)}
    # a block is read once for each (query, kv head) that lists it, but no more than the cache holds of it
    picked = [min(b, c["count"]) for b in seen_blocks]
    held, at = 0, 0
    for n, m in zip(blocks, news):
        held += min(n, sum(picked[at:at + m]))
        at += m
    return {"bytes": held * kv * (2 * bs * dim + 8) + 2 * rows + t * kv * c["count"] * 4,
            "flops": 4 * heads * dim * bs * sum(picked)}


def _codes(shape, g):
    """Codes as blocks of a trained model's keys and values have them: normal, the largest near the end of the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // max(1, out[0].numel()))
    for i in range(0, shape[0], step):
        part = out[i:i + step]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(30.0).round_().clamp_(-127, 127))
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    lens, news = _lengths(c)
    kv, dim, bs, dt = c["kv_heads"], c["dim"], c["block"], TYPES[c["dtype"]]
    blocks = [-(-n // bs) for n in lens]
    keep = blocks
    if c["op"] == "append":  # only the blocks that the call writes are in the pool, the others' places in the table are holes
        keep = [b - max(0, n - m) // bs for b, n, m in zip(blocks, lens, news)]
    pool = sum(keep) + 3
    ids = list(range(pool))
    r.shuffle(ids)
    wide = max(1, max(blocks))
    table, at = [], 0
    for b, k in zip(blocks, keep):
        table.append([-1] * (b - k) + ids[at:at + k] + [-1] * (wide - b))
        at += k
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    offsets = [0]
    for m in news:
        offsets.append(offsets[-1] + m)
    s = {"case": c, "table": ints(table), "lengths": ints(lens), "news": ints(news), "tokens": offsets[-1],
         "offsets": ints(offsets) if c["new"] > 1 else None, "max_new": max(news), "wide": wide}
    s["first"] = s["lengths"] - s["news"]  # position of the call's first token
    s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["news"].long())
    s["at"] = torch.arange(s["tokens"], device="cuda") - ints(offsets)[s["seq"]]
    s["k"] = _codes((pool, kv, bs, dim), g)
    s["v"] = _codes((pool, kv, dim, bs), g)
    s["scale"] = torch.exp2(torch.randint(-7, -4, (pool, kv, 2), generator=g, device="cuda").float())
    if c["op"] == "append":  # behind the sequence's end a block holds zeros
        held = torch.zeros(pool, dtype=torch.int64, device="cuda")
        first = [max(0, n - m) for n, m in zip(lens, news)]
        tail = [(table[b][f // bs], f % bs) for b, f in enumerate(first) if f // bs < blocks[b]]
        if tail:
            held[torch.tensor([p for p, _ in tail], device="cuda")] = torch.tensor([o for _, o in tail], device="cuda")
        slot = torch.arange(bs, device="cuda") < held[:, None]
        s["k"] *= slot[:, None, :, None]
        s["v"] *= slot[:, None, None, :]
        # keys and values as a projection leaves them: side by side in one row
        rows = torch.randn((s["tokens"], 2, kv, dim), generator=g, device="cuda")
        rows *= torch.exp(0.3 * torch.randn((1, 2, kv, dim), generator=g, device="cuda"))
        s["new_kv"] = rows.to(dt)
        s["spare"] = ids[-1]  # in no sequence's table
    s["bound"] = torch.stack((s["k"].amax(2), s["k"].amin(2)), 2)
    if c["op"] != "append":
        s["q"] = torch.randn((s["tokens"], c["heads"], dim), generator=g, device="cuda").to(dt)
    if c["op"] == "sparse":  # lists as a selection gives them: distinct, ascending, the newest block among them
        seen = (s["first"][s["seq"]] + s["at"]).clamp(min=-1) // bs + 1
        n = c["count"]
        order = torch.rand((s["tokens"], kv, wide), generator=g, device="cuda")
        j = torch.arange(wide, device="cuda")
        order = torch.where(j < seen[:, None, None], order + 2.0 * (j >= seen[:, None, None] - c["recent"]), -1.0)
        top, idx = torch.topk(order, min(n, wide), dim=-1)
        idx = torch.where(top < 0, wide, idx).sort(dim=-1).values
        idx = torch.where(idx == wide, -1, idx)
        s["lists"] = torch.nn.functional.pad(idx, (0, n - idx.shape[-1]), value=-1).to(torch.int32)
    if own:
        from dance_amd import kv as ops
        s["cache"] = ops.KVCache(s["k"], s["v"], s["scale"], s["bound"])
    return s


def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _values(s, k, v, scale):
    """What the codes stand for."""
    return {"k": k * scale[..., 0, None, None], "v": v * scale[..., 1, None, None], "scale": scale,
            "bound": s["bound"] * scale[..., 0, None, None]}


# The framework's calls.

def _own_append(s):
    from dance_amd import kv as ops
    ops.append(s["cache"], s["new_kv"][:, 0], s["new_kv"][:, 1], s["table"], s["lengths"], s["offsets"],
               max_tokens=s["max_new"])
    return _values(s, s["k"], s["v"], s["scale"])


def _own_attention(s):
    from dance_amd import kv as ops
    return ops.attention(s["cache"], s["q"], s["table"], s["lengths"], s["offsets"], max_tokens=s["max_new"],
                         return_lse=s["case"]["lse"])


def _own_select(s):
    from dance_amd import kv as ops
    c = s["case"]
    return ops.select(s["cache"], s["q"], s["table"], s["lengths"], c["count"], s["offsets"], sink=c["sink"],
                      recent=c["recent"])


def _own_sparse(s):
    from dance_amd import kv as ops
    return ops.sparse_attention(s["cache"], s["q"], s["lists"], s["table"], s["lengths"], s["offsets"])


# The plain forms.

def _exponent(a):
    """Least e with a <= 127 * 2**e, and no less than LEAST."""
    m, e = torch.frexp(a)
    return torch.where(a > 0, e - 7 + (m > 127 / 128).int(), LEAST).clamp(min=LEAST)


def _plain_append(s):
    c = s["case"]
    bs, kv, dim = c["block"], c["kv_heads"], c["dim"]
    per = (s["max_new"] + bs - 2) // bs + 1  # blocks that a sequence's new tokens may touch
    first = s["first"].clamp(min=0)
    begin = first // bs
    logical = begin[:, None] + torch.arange(per, device="cuda")
    wrote = logical * bs < s["lengths"][:, None]  # (sequence, its touched block)
    ids = s["table"].gather(1, logical.clamp(max=s["wide"] - 1).long())
    wrote &= ids >= 0
    ids = torch.where(wrote, ids, s["spare"]).long()
    pos = s["first"][s["seq"]] + s["at"]
    cell = torch.where(pos >= 0, s["seq"] * per + pos // bs - begin[s["seq"]], c["seqs"] * per)
    held = (first[:, None] - logical * bs).clamp(0, bs)  # tokens the block had
    slot = torch.arange(bs, device="cuda")
    fresh = torch.zeros((c["seqs"] * per + 1, bs), dtype=torch.bool, device="cuda")
    fresh[cell, pos % bs] = True
    fresh = fresh[:-1].view(c["seqs"], per, 1, bs, 1)
    old = (slot < held[..., None]).view(c["seqs"], per, 1, bs, 1)
    scale = s["scale"][ids]  # [sequence, block, head, 2]
    wrote = wrote[:, :, None, None, None]
    made, grown = [], []
    for i, codes in ((0, s["k"][ids]), (1, s["v"][ids].transpose(-1, -2))):
        x = torch.zeros((c["seqs"] * per + 1, bs, kv, dim), device="cuda")
        x[cell, pos % bs] = s["new_kv"][:, i].float()
        x = x[:-1].view(c["seqs"], per, bs, kv, dim).transpose(2, 3)
        was = torch.where(held[..., None] > 0, scale[..., i], 0.0)
        now = torch.maximum(was, torch.exp2(_exponent(x.abs().amax((-1, -2))).float()))
        kept = torch.where(old, (codes * (was / now)[..., None, None]).round(), 0.0)
        made.append(torch.where(wrote, torch.where(fresh, (x / now[..., None, None]).round(), kept).to(torch.int8), codes))
        grown.append(now)
    live = (old | fresh).expand(made[0].shape)
    bound = torch.stack((torch.where(live, made[0], -128).amax(3), torch.where(live, made[0], 127).amin(3)), 3)
    s["bound"][ids] = torch.where(wrote, bound, s["bound"][ids])
    s["k"][ids] = made[0]
    s["v"][ids] = made[1].transpose(-1, -2)
    s["scale"][ids] = torch.where(wrote[..., 0], torch.stack(grown, -1), scale)
    return _values(s, s["k"], s["v"], s["scale"])


def _softmax_products(logits, v):
    """(sum of weights * v, log of the weights' sum) over the last axis of the logits; 0 and -inf where all are masked."""
    m = logits.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(logits - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o, (m + torch.log(total)).squeeze(-1)


def _plain_attention(s):
    c = s["case"]
    kv, dim, bs, n, seqs = c["kv_heads"], c["dim"], c["block"], s["max_new"], c["seqs"]
    group = c["heads"] // kv
    safe = s["table"].clamp(min=0).long()
    scale = s["scale"][safe]
    k = (s["k"][safe] * scale[..., 0, None, None]).transpose(1, 2).reshape(seqs, kv, -1, dim)
    v = (s["v"][safe] * scale[..., 1, None, None]).permute(0, 2, 1, 4, 3).reshape(seqs, kv, -1, dim)
    q = torch.zeros((seqs, n, c["heads"], dim), device="cuda")
    q[s["seq"], s["at"]] = s["q"].float()
    q = q.view(seqs, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * n, dim)
    logits = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(dim ** -0.5).view(seqs, kv, group, n, -1)
    pos = s["first"][:, None] + torch.arange(n, device="cuda")
    hidden = torch.arange(k.shape[2], device="cuda") > pos[..., None]
    logits.masked_fill_(hidden[:, None, None], -math.inf)
    o, lse = _softmax_products(logits.view(seqs, kv, group * n, -1), v)
    o = o.view(seqs, kv, group, n, dim).permute(0, 3, 1, 2, 4).reshape(seqs, n, c["heads"], dim)
    o = o[s["seq"], s["at"]].to(TYPES[c["dtype"]])
    if not c["lse"]:
        return o
    return o, lse.view(seqs, kv, group, n).permute(0, 3, 1, 2).reshape(seqs, n, c["heads"])[s["seq"], s["at"]]


def _plain_select(s):
    c = s["case"]
    kv, dim, bs, t, wide = c["kv_heads"], c["dim"], c["block"], s["tokens"], s["wide"]
    group = c["heads"] // kv
    q = s["q"].float()
    e = _exponent(q.abs().amax(-1))
    q = (q * torch.exp2(-e.float())[..., None]).round()
    safe = s["table"].clamp(min=0).long()
    bound = s["bound"][safe].float().permute(0, 2, 3, 4, 1).reshape(c["seqs"], kv, 2 * dim, wide)
    # the larger product of a dimension is that with the largest code for positive q, the least for negative q
    both = torch.cat((q.clamp(min=0), q.clamp(max=0)), -1)
    n = s["max_new"]
    rows = torch.zeros((c["seqs"], n, c["heads"], 2 * dim), device="cuda")
    rows[s["seq"], s["at"]] = both
    rows = rows.view(c["seqs"], n, kv, group, 2 * dim).transpose(1, 2).reshape(c["seqs"], kv, n * group, 2 * dim)
    score = torch.matmul(rows, bound).view(c["seqs"], kv, n, group, wide).transpose(1, 2)[s["seq"], s["at"]]
    score = score * s["scale"][safe][..., 0].transpose(1, 2)[s["seq"]][:, :, None]
    score = (score * torch.exp2(e.float()).view(t, kv, group, 1)).amax(2)
    seen = ((s["first"][s["seq"]] + s["at"]).clamp(min=-1) // bs + 1)[:, None, None]
    j = torch.arange(wide, device="cuda")
    score = torch.where((j < c["sink"]) | (j >= seen - c["recent"]), math.inf, score)
    score = torch.where(j < seen, score, -math.inf)
    score, order = torch.sort(score, dim=-1, descending=True, stable=True)
    order = torch.where(score == -math.inf, wide, order)[..., :c["count"]].sort(dim=-1).values
    order = torch.where(order == wide, -1, order)
    return torch.nn.functional.pad(order, (0, c["count"] - order.shape[-1]), value=-1).to(torch.int32)


def _plain_sparse(s):
    c = s["case"]
    kv, dim, bs, t = c["kv_heads"], c["dim"], c["block"], s["tokens"]
    lists = s["lists"].long()
    ids = s["table"][s["seq"][:, None, None], lists.clamp(min=0)].long()
    ids, head = ids.clamp(min=0), torch.arange(kv, device="cuda")[None, :, None]
    scale = s["scale"][ids, head]
    k = (s["k"][ids, head] * scale[..., 0, None, None]).reshape(t, kv, -1, dim)
    v = (s["v"][ids, head] * scale[..., 1, None, None]).transpose(-1, -2).reshape(t, kv, -1, dim)
    q = s["q"].float().view(t, kv, -1, dim)
    logits = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(dim ** -0.5)
    pos = (s["first"][s["seq"]] + s["at"])[:, None, None, None]
    shown = (lists[..., None] >= 0) & (lists[..., None] * bs + torch.arange(bs, device="cuda") <= pos)
    logits.masked_fill_(~shown.view(t, kv, 1, -1), -math.inf)
    return _softmax_products(logits, v)[0].reshape(t, c["heads"], dim).to(TYPES[c["dtype"]])


_own = {"append": _own_append, "attention": _own_attention, "select": _own_select, "sparse": _own_sparse}
_plain = {"append": _plain_append, "attention": _plain_attention, "select": _plain_select, "sparse": _plain_sparse}


# The definitions in 64 bits, sequence by sequence.

def _scale64(a):
    return 2.0 ** max(LEAST, math.ceil(math.log2(a / 127.0))) if a > 0 else 2.0 ** LEAST


def _attend64(q, k, v, shown):
    """q [rows, dim], k and v [tokens, dim], shown [rows, tokens] -> (o, lse)."""
    logits = (q @ k.T) / math.sqrt(q.shape[1])
    logits[~shown] = -math.inf
    lse = torch.logsumexp(logits, 1)
    o = torch.exp(logits - torch.where(torch.isinf(lse), 0.0, lse)[:, None]) @ v
    return o, lse


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    lens, news = _lengths(c)
    kv, dim, bs = c["kv_heads"], c["dim"], c["block"]
    group = c["heads"] // kv
    table = s["table"].tolist()
    if c["op"] == "append":
        if sum(news) * kv > 1 << 21:
            return None
        val = [s["k"].double() * s["scale"][:, :, 0, None, None].double(),
               (s["v"].double() * s["scale"][:, :, 1, None, None].double()).transpose(2, 3)]
        scale, bound, at = s["scale"].double().cpu(), s["bound"].double().cpu() * s["scale"].double().cpu()[:, :, 0, None, None], 0
        for b, (n, m) in enumerate(zip(lens, news)):
            x = s["new_kv"][at:at + m].double()
            at += m
            for j in range(max(0, n - m) // bs, -(-n // bs)):
                p, lo, hi = table[b][j], max(n - m, j * bs), min(n, (j + 1) * bs)
                part, old = x[lo - (n - m):hi - (n - m)], lo - j * bs
                top = part.abs().amax((0, 3)).tolist()
                for i in range(2):
                    for h in range(kv):
                        step = max(_scale64(top[i][h]), float(scale[p, h, i]) if old else 0.0)
                        block = val[i][p, h]
                        block[:old] = torch.round(block[:old] / step) * step
                        block[old:old + hi - lo] = torch.round(part[:, i, h] / step) * step
                        block[old + hi - lo:] = 0
                        scale[p, h, i] = step
                        if i == 0:
                            live = block[:old + hi - lo]
                            bound[p, h] = torch.stack((live.amax(0), live.amin(0))).cpu()
        return {"k": val[0], "v": val[1].transpose(2, 3), "scale": scale, "bound": bound}
    out, sums, picks, at = [], [], [], 0
    scale = s["scale"].double()
    for b, (n, m) in enumerate(zip(lens, news)):
        q = s["q"][at:at + m].double()
        pos = torch.arange(n - m, n, device="cuda")
        ids = torch.tensor(table[b][:-(-n // bs)], dtype=torch.int64, device="cuda")
        if c["op"] == "attention":
            o, l = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
            for h in range(kv):
                k = (s["k"][ids, h].double() * scale[ids, h, 0, None, None]).reshape(-1, dim)
                v = (s["v"][ids, h].double() * scale[ids, h, 1, None, None]).transpose(1, 2).reshape(-1, dim)
                shown = torch.arange(len(k), device="cuda") <= pos[:, None]
                for f in range(h * group, (h + 1) * group):
                    o[:, f], l[:, f] = _attend64(q[:, f], k, v, shown)
            out.append(o)
            sums.append(l)
        elif c["op"] == "select":
            top = q.abs().amax(2)
            step = torch.tensor([[_scale64(a) for a in row] for row in top.tolist()], dtype=torch.float64, device="cuda")
            rounded = torch.round(q / step[:, :, None])
            got = torch.full((m, kv, c["count"]), -1, dtype=torch.int32, device="cuda")
            if m * c["heads"] * len(ids) > 1 << 26:
                return None
            for h in range(kv):
                hi, lo = s["bound"][ids, h, 0].double(), s["bound"][ids, h, 1].double()
                score = torch.full((m, len(ids)), -math.inf, dtype=torch.float64, device="cuda")
                for f in range(h * group, (h + 1) * group):
                    r = rounded[:, f]
                    one = (r * (r > 0)) @ hi.T + (r * (r < 0)) @ lo.T
                    score = torch.maximum(score, one * scale[ids, h, 0] * step[:, f, None])
                j = torch.arange(len(ids), device="cuda")
                seen = torch.clamp(pos, min=-1)[:, None] // bs + 1
                score[(j < c["sink"]) | (j >= seen - c["recent"])] = math.inf
                score[j >= seen] = -math.inf
                order = torch.argsort(score, dim=1, descending=True, stable=True)[:, :c["count"]]
                order[~(torch.gather(score, 1, order) > -math.inf)] = 1 << 30
                order = order.sort(dim=1).values
                got[:, h, :order.shape[1]] = torch.where(order == 1 << 30, -1, order).int()
            picks.append(got)
        else:
            if s["tokens"] * kv > 20000:
                return None
            o = torch.zeros_like(q)
            for i in range(m):
                for h in range(kv):
                    chosen = s["lists"][at + i, h]
                    chosen = chosen[chosen >= 0].long()
                    if len(chosen):
                        p = ids[chosen]
                        k = (s["k"][p, h].double() * scale[p, h, 0, None, None]).reshape(-1, dim)
                        v = (s["v"][p, h].double() * scale[p, h, 1, None, None]).transpose(1, 2).reshape(-1, dim)
                        where = (chosen[:, None] * bs + torch.arange(bs, device="cuda")).reshape(1, -1)
                        f = slice(h * group, (h + 1) * group)
                        o[i, f] = _attend64(q[i, f], k, v, (where <= pos[i]).expand(group, -1))[0]
            out.append(o)
        at += m
    if c["op"] == "select":
        return torch.cat(picks)
    return (torch.cat(out), torch.cat(sums)) if c["lse"] else torch.cat(out)
