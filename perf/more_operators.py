"""The calls that the speed of the cache's further operators is measured on.

Blocks of the key-value cache have owners: sequences that fork share them, grow
and shrink (`pages`), blocks are copied for all layers at once (`copy`), chosen
tokens move to dense blocks (`compact`). Rows attend to all tokens of another
sequence, an encoder's or a prefix that many share (`cross`), and attentions over
parts of a context are joined (`join`). `run` computes them in plain torch
operations, or with the framework's kernels where `own` is set.

A cache: `blocks` of `block` tokens; for each block and kv head the codes of
its keys (tokens x dim) and values (dim x tokens), a scale for each of the two,
and the largest and least key code for each dimension. `table` gives the block
of each part of a sequence, `lengths` the sequences' tokens. `refs` counts each
block's places in the table.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEAST = -100  # exponent of the least scale


def _case(name, op, **more):
    c = {"op": op, **more}
    return {"name": name, **c} if name else c


def _pages(name, users, beams, block, least, most, grow, back, idle=0, spare=0.25):
    return _case(name, "pages", users=users, beams=beams, block=block, least=least, most=most, grow=grow, back=back,
                 idle=idle, spare=spare)


def _copy(name, layers, kv_heads, dim, block, pairs, real):
    return _case(name, "copy", layers=layers, kv_heads=kv_heads, dim=dim, block=block, pairs=pairs, real=real)


def _compact(name, seqs, kv_heads, dim, block, least, most, share, same=False):
    return _case(name, "compact", seqs=seqs, kv_heads=kv_heads, dim=dim, block=block, least=least, most=most, share=share,
                 same=same)


def _cross(name, dtype, seqs, heads, kv_heads, dim, block, least, most, new=1, ragged=False, idle=0, lse=False):
    return _case(name, "cross", dtype=dtype, seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, block=block, least=least,
                 most=most, new=new, ragged=ragged, idle=idle, lse=lse)


def _join(name, dtype, tokens, heads, dim, parts, some=False, lse=False):
    return _case(name, "join", dtype=dtype, tokens=tokens, heads=heads, dim=dim, parts=parts, some=some, lse=lse)


def listed():
    return [
        # a step of a beam search: the beams of each user are chosen anew and grow by a token
        _pages("beam_step", 8, 4, 64, 300, 2500, 1, 0),
        # a large batch with drafts of eight tokens of which some are given back, small blocks, long tables
        _pages("draft_batch", 128, 4, 32, 500, 60000, 8, 5, idle=3),
        # the shared last blocks of some forked sequences, in all layers
        _copy("copy_tails", 16, 8, 128, 64, 64, 16),
        # whole sequences to another pool
        _copy("copy_pool", 16, 8, 128, 64, 600, 600),
        # a few short sequences of odd lengths, small blocks, 96 dimensions
        _compact("evict_odd", 3, 5, 96, 16, 100, 4000, 0.4),
        # half of the tokens of a batch go, other ones for each head
        _compact("evict_half", 16, 8, 128, 64, 4000, 24000, 0.5),
        # a long context keeps every fiftieth token
        _compact("evict_long", 1, 8, 128, 64, 262144, 262144, 0.02),
        # a decoder's step over its encoder's states, as many kv heads as heads
        _cross("cross_step", "bf16", 48, 16, 16, 64, 64, 200, 1500, idle=1),
        # all rows of decoders over their encoders' states, of different numbers
        _cross("cross_rows", "f16", 6, 20, 20, 64, 64, 700, 1500, new=448, ragged=True),
        # a step of 64 sequences that share a long prompt: the part of it
        _cross("prefix_batch", "bf16", 1, 32, 8, 128, 64, 40000, 40000, new=64, lse=True),
        # that part and each sequence's own
        _join("join_step", "bf16", 64, 32, 128, 2),
        # three parts for a chunk's rows, two of them for some of the rows only
        _join("join_chunk", "f16", 8192, 32, 128, 3, some=True, lse=True),
    ]


def _log(rng, a, b):
    return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        key = c["op"]
        most[key] = {k: max(most.get(key, {}).get(k, 0), w[k]) for k in w}
    while True:
        op = rng.choice(["pages", "copy", "compact", "compact", "cross", "cross", "join"])
        kv = rng.choice([1, 2, 3, 4, 5, 8, 8, 12, 16])
        dim = rng.choice([64, 96, 128, 128, 192, 256])
        block = rng.choice([16, 32, 64, 64, 128])
        if op == "pages":
            users, beams = _log(rng, 1, 200), rng.choice([1, 2, 3, 4, 5, 8])
            grow = rng.choice([1, 1, 2, 5, 8]) if rng.random() < 0.7 else _log(rng, 10, 2000)
            longest = _log(rng, 8, 60000)
            c = _pages(None, users, beams, block, _log(rng, 1, longest), longest, grow, rng.randint(0, grow),
                       idle=rng.choice([0, 0, 1]) if users > 1 else 0, spare=rng.choice([0.05, 0.25, 1.0]))
            if users * beams * ((longest + grow) // block + 2) > 1 << 20:
                continue
        elif op == "copy":
            pairs = _log(rng, 1, 600)
            c = _copy(None, rng.choice([1, 2, 5, 16, 24, 32]), kv, dim, block, pairs, rng.randint(1, pairs))
        elif op == "compact":
            longest = _log(rng, 8, 262144)
            c = _compact(None, _log(rng, 1, 64), kv, dim, block, _log(rng, max(1, longest // 8), longest), longest,
                         rng.choice([0.02, 0.1, 0.4, 0.5, 0.9, 1.0]), same=rng.random() < 0.3)
            if sum(_tokens(c)) * kv * dim > 1 << 29:
                continue
        elif op == "cross":
            group = rng.choice([1, 1, 2, 3, 4, 4, 5, 8, 16])
            longest = _log(rng, 8, 60000)
            new = rng.choice([1, 1, 1, 4]) if rng.random() < 0.5 else _log(rng, 2, 1000)
            c = _cross(None, rng.choice(["bf16", "f16"]), _log(rng, 1, 64), kv * group, kv, dim, block,
                       _log(rng, max(1, longest // 8), longest), longest, new=new, ragged=new > 1 and rng.random() < 0.6,
                       lse=rng.random() < 0.4)
            lens, news = _lengths(c)
            if c["heads"] * c["seqs"] * max(news) * (max(lens) + block) > 1 << 30 or kv * dim * c["seqs"] * max(lens) > 1 << 30:
                continue
            if c["seqs"] > 1 and rng.random() < 0.3:
                c["idle"] = 1
        else:
            c = _join(None, rng.choice(["bf16", "f16"]), _log(rng, 1, 8192), kv * rng.choice([1, 2, 4]), dim,
                      rng.choice([2, 2, 3, 4, 8]), some=rng.random() < 0.4, lse=rng.random() < 0.5)
        w = work(c)
        if all(w[k] <= most[op][k] for k in w) and w["bytes"] > 2000:
            return c


def _rand(c):
    return random.Random(" ".join("%s=%s" % kv for kv in sorted(c.items()) if kv[0] != "name"))


def _tokens(c):
    """Tokens of each sequence: from the case alone."""
    r = _rand(c)
    return [_log(r, c["least"], c["most"]) for _ in range(c["seqs"])]


def _lengths(c):
    """Tokens of each sequence, and how many rows read them."""
    r = _rand({**c, "idle": 0})
    lens = [_log(r, c["least"], c["most"]) for _ in range(c["seqs"])]
    news = [_log(r, 1, c["new"]) if c["ragged"] else c["new"] for _ in lens]
    for b in range(c["idle"]):  # slots of the batch that hold no sequence: a row each, nothing to read
        lens[b], news[b] = 0, 1
    return lens, news


def _counts(c):
    return [max(1, round(n * c["share"])) for n in _tokens(c)]


def work(case):
    c = case
    if c["op"] == "pages":
        seqs = c["users"] * c["beams"]
        lens = [n for u in _beams(c) for n in u[1]]
        width, blocks = _room(c)
        places = sum(-(-n // c["block"]) for n in lens)
        return {"bytes": 8 * places + 4 * blocks + 40 * seqs, "flops": 0}
    if c["op"] == "copy":
        return {"bytes": 2 * c["real"] * c["layers"] * c["kv_heads"] * (2 * c["dim"] * (c["block"] + 1) + 8) + 8 * c["pairs"],
                "flops": 0}
    if c["op"] == "compact":
        counts = _counts(c)
        blocks = sum(-(-n // c["block"]) for n in counts)
        lists = sum(counts) * 4 * (1 if c["same"] else c["kv_heads"])
        kv, dim = c["kv_heads"], c["dim"]
        return {"bytes": sum(counts) * kv * dim * 2 + blocks * kv * (2 * dim * c["block"] + 2 * dim + 8) + lists, "flops": 0}
    if c["op"] == "cross":
        lens, news = _lengths(c)
        blocks, t = sum(-(-n // c["block"]) for n in lens), sum(news)
        return {"bytes": sum(lens) * c["kv_heads"] * c["dim"] * 2 + blocks * c["kv_heads"] * 8
                + t * c["heads"] * (c["dim"] * 4 + (4 if c["lse"] else 0)),
                "flops": 4 * c["heads"] * c["dim"] * sum(n * m for n, m in zip(lens, news))}
    rows = c["tokens"] * c["heads"]
    read = sum(c["tokens"] if not i or not c["some"] else -(-c["tokens"] // 2) for i in range(c["parts"])) * c["heads"]
    return {"bytes": read * (c["dim"] * 2 + 4) + rows * (c["dim"] * 2 + (4 if c["lse"] else 0)),
            "flops": 2 * read * c["dim"]}


# ----------------------------------------------------------------- inputs

def _beams(c):
    """For each user the tokens that its beams share and the tokens of each beam."""
    r = _rand(c)
    out = []
    for u in range(c["users"]):
        n = _log(r, c["least"], c["most"])
        if u < c["idle"]:
            out.append((0, [0] * c["beams"]))
        else:  # the beams of a search are equally long
            out.append((r.randint(0, n), [n] * c["beams"]))
    return out


def _room(c):
    """Places of a table row, and blocks of the pool."""
    bs, lens = c["block"], [n for u in _beams(c) for n in u[1]]
    width = max(lens) // bs + c["grow"] // bs + 3
    used = sum(s // bs + sum(-(-n // bs) - s // bs for n in ns) for s, ns in _beams(c))
    return width, int(used * (1 + c["spare"])) + 2 + int(c["spare"] * c["grow"] / bs * len(lens))


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _prepare_pages(c, seed):
    r = random.Random(seed)
    bs, seqs, beams = c["block"], c["users"] * c["beams"], c["beams"]
    width, blocks = _room(c)
    ids = list(range(blocks))
    r.shuffle(ids)
    at, rows, lens, parents, refs = 0, [], [], [], [0] * blocks
    for u, (shared, ns) in enumerate(_beams(c)):
        head = ids[at:at + shared // bs]
        at += len(head)
        for n in ns:
            tail = ids[at:at + -(-n // bs) - len(head)]
            at += len(tail)
            rows.append(head + tail + [-1] * (width - len(head) - len(tail)))
            lens.append(n)
        # the beams that go on, each user's own: some twice, some not at all; now and then a slot ends
        parents += [u * beams + r.randrange(beams) if r.random() > 0.02 else -1 for _ in range(beams)]
    for row in rows:
        for p in row:
            if p >= 0:
                refs[p] += 1
    after = [lens[p] if p >= 0 else 0 for p in parents]
    upto = [n + c["grow"] if p >= 0 and n else n for p, n in zip(parents, after)]
    s = {"case": c, "parents": _ints(parents), "upto": _ints(upto), "keep": _ints([n - c["back"] if m < n else n
                                                                               for m, n in zip(after, upto)]),
         "table": _ints(rows), "lengths": _ints(lens), "kept": _ints(refs)}
    s["refs"] = s["kept"].clone()  # a pass starts from the same owners
    if own:
        from dance_amd import kv as ops
        s["pages"] = ops.Pages(s["refs"], bs)
    return s


def _codes(shape, g):
    """Codes as blocks of a trained model's keys and values have them: normal, the largest near the end of the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(30.0).round_().clamp_(-127, 127))
    return out


def _pool(layers, blocks, kv, dim, bs, g):
    p = {"k": _codes((layers, blocks, kv, bs, dim), g), "v": _codes((layers, blocks, kv, dim, bs), g),
         "scale": torch.exp2(torch.randint(-7, -4, (layers, blocks, kv, 2), generator=g, device="cuda").float())}
    p["bound"] = torch.stack((p["k"].amax(3), p["k"].amin(3)), 3)
    return p


def _empty(layers, blocks, kv, dim, bs):
    z = lambda *s: torch.zeros((layers, blocks, kv, *s), dtype=torch.int8, device="cuda")  # noqa: E731
    return {"k": z(bs, dim), "v": z(dim, bs), "scale": torch.ones((layers, blocks, kv, 2), device="cuda"), "bound": z(2, dim)}


def _caches(p):
    from dance_amd import kv as ops
    return [ops.KVCache(*(p[x][i] for x in ("k", "v", "scale", "bound"))) for i in range(len(p["k"]))]


def _values(p):
    """What the codes stand for: a code of seven bits and a sign times a power of two is exact in bfloat16."""
    s = p["scale"].bfloat16()
    return {"k": p["k"] * s[..., 0, None, None], "v": p["v"] * s[..., 1, None, None], "scale": p["scale"],
            "bound": p["bound"] * s[..., 0, None, None]}


def _prepare_copy(c, seed):
    g, r = torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    n, dims = c["pairs"], (c["kv_heads"], c["dim"], c["block"])
    src, dst = [r.randrange(c["real"] + 3) for _ in range(n)], list(range(c["real"] + 1))
    r.shuffle(dst)
    real = sorted(r.sample(range(n), c["real"]))
    at = {i: j for j, i in enumerate(real)}
    s = {"case": c, "from": _pool(c["layers"], c["real"] + 3, *dims, g), "to": _empty(c["layers"], c["real"] + 1, *dims),
         "src": _ints([src[i] if i in at else -1 for i in range(n)]),
         "dst": _ints([dst[at[i]] if i in at else -1 for i in range(n)])}
    if own:
        s["caches"], s["into"] = _caches(s["from"]), _caches(s["to"])
    return s


def _prepare_compact(c, seed):
    g, r = torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    kv, dim, bs, lens, counts = c["kv_heads"], c["dim"], c["block"], _tokens(c), _counts(c)

    def tables(ns, extra):
        need = [-(-n // bs) for n in ns]
        ids = list(range(sum(need) + extra))
        r.shuffle(ids)
        rows, at = [], 0
        for n in need:
            rows.append(ids[at:at + n] + [-1] * (max(need) - n))
            at += n
        return _ints(rows), len(ids), ids[-1]

    table, pool, _ = tables(lens, 2)
    into_table, into, spare = tables(counts, 1)
    most = max(counts)
    keep = torch.full((c["seqs"], 1 if c["same"] else kv, most), -1, dtype=torch.int32, device="cuda")
    for b, (n, m) in enumerate(zip(lens, counts)):  # tokens of some importance: distinct, in their order
        for h in range(keep.shape[1]):
            weight = torch.rand(n, generator=g, device="cuda")
            weight[max(0, n - m // 8):] += 1  # the newest stay
            keep[b, h, :m] = torch.topk(weight, m).indices.sort().values.int()
    s = {"case": c, "from": _pool(1, pool, kv, dim, bs, g), "to": _empty(1, into, kv, dim, bs), "table": table,
         "into_table": into_table, "lengths": _ints(lens), "counts": _ints(counts), "keep": keep, "most": most,
         "spare": spare}  # a block of no sequence
    if own:
        s["cache"], s["into"] = _caches(s["from"])[0], _caches(s["to"])[0]
    return s


def _prepare_cross(c, seed):
    g, r = torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    lens, news = _lengths(c)
    bs = c["block"]
    blocks = [-(-n // bs) for n in lens]
    ids = list(range(sum(blocks) + 2))
    r.shuffle(ids)
    rows, at, offsets = [], 0, [0]
    for n, m in zip(blocks, news):
        rows.append(ids[at:at + n] + [-1] * (max(max(blocks), 1) - n))
        at += n
        offsets.append(offsets[-1] + m)
    s = {"case": c, "table": _ints(rows), "lengths": _ints(lens), "offsets": _ints(offsets) if c["new"] > 1 else None,
         "news": news, "max_new": max(news), **{k: v[0] for k, v in _pool(1, len(ids), c["kv_heads"], c["dim"], bs, g).items()}}
    s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), _ints(news).long())
    s["at"] = torch.arange(offsets[-1], device="cuda") - _ints(offsets)[s["seq"]]
    s["q"] = torch.randn((offsets[-1], c["heads"], c["dim"]), generator=g, device="cuda").to(TYPES[c["dtype"]])
    if own:
        from dance_amd import kv as ops
        s["cache"] = ops.KVCache(s["k"], s["v"], s["scale"], s["bound"])
    return s


def _prepare_join(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, heads = c["tokens"], c["heads"]
    s = {"case": c, "parts": [], "lses": [], "rows": []}
    for i in range(c["parts"]):
        n = t if not i or not c["some"] else -(-t // 2)
        rows = None
        if n < t:  # a part that only some of the rows have, in another order
            where = torch.randperm(t, generator=g, device="cuda")[:n]
            rows = torch.full((t,), -1, dtype=torch.int32, device="cuda")
            rows[where] = torch.arange(n, dtype=torch.int32, device="cuda")
        s["rows"].append(rows)
        s["parts"].append(torch.randn((n, heads, c["dim"]), generator=g, device="cuda").to(TYPES[c["dtype"]]))
        lse = 6 + 2 * torch.randn((n, heads), generator=g, device="cuda")
        s["lses"].append(lse.masked_fill_(torch.rand(lse.shape, generator=g, device="cuda") < 0.03, -math.inf))
    return s


def prepare(case, seed):
    return {"pages": _prepare_pages, "copy": _prepare_copy, "compact": _prepare_compact, "cross": _prepare_cross,
            "join": _prepare_join}[case["op"]](case, seed)


def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


# The framework's calls.

def _own_pages(s):
    from dance_amd import kv as ops
    s["refs"].copy_(s["kept"])
    table, lengths = ops.fork(s["pages"], s["table"], s["lengths"], s["parents"])
    now, src, dst = ops.reserve(s["pages"], table, lengths, s["upto"])
    ops.release(s["pages"], table, lengths, keep=s["keep"])
    return {"table": table, "lengths": lengths, "refs": s["refs"], "now": now, "src": src, "dst": dst}


def _own_copy(s):
    from dance_amd import kv as ops
    ops.copy(s["caches"], s["src"], s["dst"], into=s["into"])
    return _values(s["to"])


def _own_compact(s):
    from dance_amd import kv as ops
    ops.compact(s["cache"], s["keep"], s["counts"], s["table"], s["lengths"], s["into_table"], into=s["into"])
    return _values(s["to"])


def _own_cross(s):
    from dance_amd import kv as ops
    return ops.cross_attention(s["cache"], s["q"], s["table"], s["lengths"], s["offsets"], max_tokens=s["max_new"],
                               return_lse=s["case"]["lse"])


def _own_join(s):
    from dance_amd import kv as ops
    return ops.join(s["parts"], s["lses"], s["rows"] if s["case"]["some"] else None, return_lse=s["case"]["lse"])


# The plain forms.

def _plain_pages(s):
    c = s["case"]
    bs, blocks = c["block"], s["refs"].numel()
    seqs, width = s["table"].shape
    s["refs"].copy_(s["kept"])
    aside = torch.arange(blocks, blocks + seqs * width, device="cuda")  # entries outside the pool count in places of their own
    one = torch.ones_like(aside, dtype=torch.int32)

    def count(refs, entries, sign):
        entries = entries.reshape(-1)
        ok = (entries >= 0) & (entries < blocks)
        refs.index_add_(0, torch.where(ok, entries, aside[:entries.numel()]), one[:entries.numel()] * sign)

    refs = torch.cat((s["refs"], torch.zeros_like(one)))
    # fork
    ok = (s["parents"] >= 0) & (s["parents"] < seqs)
    parents = torch.where(ok, s["parents"], 0).long()
    table = torch.where(ok[:, None], s["table"][parents], -1)
    lengths = torch.where(ok, s["lengths"][parents], 0)
    count(refs, table, 1)
    count(refs, s["table"], -1)
    # reserve: the places that need a block of their own
    upto, at = s["upto"], torch.arange(width, device="cuda")
    first = lengths // bs
    grows = (upto > lengths) & (upto <= width * bs)
    mine = grows[:, None] & (at >= first[:, None]) & (at < ((upto + bs - 1) // bs)[:, None])
    valid = (table >= 0) & (table < blocks)
    many = valid & (refs[torch.where(valid, table, blocks).long()] > 1)
    partly = (at == first[:, None]) & (lengths % bs != 0)[:, None]
    end = torch.where(mine & partly & valid, table, -1).amax(1)  # the partly filled block of a sequence that grows
    alike = (end[:, None] == end) & (end >= 0)
    later = torch.triu(alike, 1).any(1)
    last = (end >= 0) & ~later & (alike.sum(1) == refs[end.clamp(min=0).long()]) & (alike.sum(1) > 1)
    fresh = mine & torch.where(partly, many & ~last[:, None], many | ~valid)
    need = fresh.sum(1)
    upper = torch.cumsum(need, 0)
    free = refs[:blocks] == 0
    served = grows & ((upper <= free.sum()) | ((need == 0) & ~last))
    fresh &= served[:, None]
    # the blocks that nobody owns, in their order
    order = torch.cumsum(free, 0) - 1
    ids = torch.full((blocks + 1,), -1, dtype=torch.int32, device="cuda")
    ids[torch.where(free, order, blocks)] = torch.arange(blocks, dtype=torch.int32, device="cuda")
    rank = (upper - need)[:, None] + torch.cumsum(fresh, 1) - 1
    given = torch.where(fresh, ids[torch.where(fresh, rank, 0)], -1)
    copied = fresh & partly
    src, dst = torch.where(copied, table, -1).amax(1), torch.where(copied, given, -1).amax(1)
    count(refs, torch.where(fresh & valid, table, -1), -1)
    count(refs, given, 1)
    table = torch.where(fresh, given, table)
    now = torch.where(served, upto, torch.where(upto <= lengths, lengths, 0))
    lengths = torch.where(served, upto, lengths)
    # release
    lengths = torch.minimum(lengths, s["keep"].clamp(min=0))
    dropped = at >= ((lengths + bs - 1) // bs)[:, None]
    count(refs, torch.where(dropped, table, -1), -1)
    table = torch.where(dropped, -1, table)
    s["refs"].copy_(refs[:blocks])
    return {"table": table, "lengths": lengths, "refs": s["refs"], "now": now, "src": src, "dst": dst}


def _plain_copy(s):
    live = torch.where(s["src"] >= 0, 1, 0).bool()
    src, dst = s["src"].long(), s["dst"].long()
    n = s["to"]["k"].shape[1]
    for name, to in s["to"].items():
        for i in range(len(to)):  # layer by layer; pairs that are none change nothing
            pick = torch.full((n + 1,), -1, dtype=torch.int64, device="cuda")
            pick[torch.where(live, dst, n)] = torch.where(live, src, -1)
            pick = pick[:n]
            got = s["from"][name][i][pick.clamp(min=0)]
            to[i] = torch.where((pick >= 0).view(-1, *[1] * (got.ndim - 1)), got, to[i])
    return _values(s["to"])


def _exponent(a):
    """Least e with a <= 127 * 2**e, and no less than LEAST."""
    m, e = torch.frexp(a)
    return torch.where(a > 0, e - 7 + (m > 127 / 128).int(), LEAST).clamp(min=LEAST)


def _plain_compact(s):
    c = s["case"]
    kv, dim, bs, seqs = c["kv_heads"], c["dim"], c["block"], c["seqs"]
    per = s["into_table"].shape[1]
    f = {k: v[0] for k, v in s["from"].items()}
    to = {k: v[0] for k, v in s["to"].items()}
    keep = torch.nn.functional.pad(s["keep"], (0, per * bs - s["most"]), value=-1).expand(-1, kv, -1)
    live = (torch.arange(per * bs, device="cuda") < s["counts"][:, None])[:, None] & (keep >= 0)
    live &= keep < s["lengths"][:, None, None]
    at = torch.where(live, keep, 0).long()
    block = s["table"].long()[torch.arange(seqs, device="cuda")[:, None, None], at // bs]
    live &= (block >= 0) & (block < len(f["k"]))
    block, head, slot = block.clamp(min=0), torch.arange(kv, device="cuda")[None, :, None], at % bs
    scale = f["scale"][block, head] * live[..., None]
    k = (f["k"][block, head, slot] * scale[..., 0, None]).view(seqs, kv, per, bs, dim)
    v = (f["v"][block, head, :, slot] * scale[..., 1, None]).view(seqs, kv, per, bs, dim)
    written = torch.arange(per, device="cuda") < (s["counts"][:, None] + bs - 1) // bs
    where = torch.where(written, s["into_table"], s["spare"]).long()
    step = [torch.exp2(_exponent(x.abs().amax((-1, -2))).float()) for x in (k, v)]
    k, v = ((x / e[..., None, None]).round().to(torch.int8) for x, e in zip((k, v), step))
    token = torch.arange(per * bs, device="cuda").view(per, bs) < s["counts"][:, None, None]
    token = token[:, None, :, :, None]
    bound = torch.stack((torch.where(token, k, -128).amax(3), torch.where(token, k, 127).amin(3)), 3)
    for name, x in (("k", k), ("v", v.transpose(-1, -2)), ("scale", torch.stack(step, -1)), ("bound", bound)):
        x = x.transpose(1, 2)  # sequence, block, head
        to[name][where] = torch.where(written.view(seqs, per, *[1] * (x.ndim - 2)), x, to[name][where])
    return _values(s["to"])


def _softmax_products(logits, v):
    """(sum of weights * v, log of the weights' sum) over the last axis of the logits; 0 and -inf where all are masked."""
    m = logits.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(logits - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o, (m + torch.log(total)).squeeze(-1)


def _plain_cross(s):
    c = s["case"]
    kv, dim, n, seqs = c["kv_heads"], c["dim"], s["max_new"], c["seqs"]
    group = c["heads"] // kv
    safe = s["table"].clamp(min=0).long()
    scale = s["scale"][safe]
    k = (s["k"][safe] * scale[..., 0, None, None]).transpose(1, 2).reshape(seqs, kv, -1, dim)
    v = (s["v"][safe] * scale[..., 1, None, None]).permute(0, 2, 1, 4, 3).reshape(seqs, kv, -1, dim)
    q = torch.zeros((seqs, n, c["heads"], dim), device="cuda")
    q[s["seq"], s["at"]] = s["q"].float()
    q = q.view(seqs, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * n, dim)
    logits = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(dim ** -0.5)
    hidden = torch.arange(k.shape[2], device="cuda") >= s["lengths"][:, None]
    logits.masked_fill_(hidden[:, None, None], -math.inf)
    o, lse = _softmax_products(logits, v)
    o = o.view(seqs, kv, group, n, dim).permute(0, 3, 1, 2, 4).reshape(seqs, n, c["heads"], dim)
    o = o[s["seq"], s["at"]].to(TYPES[c["dtype"]])
    if not c["lse"]:
        return o
    return o, lse.view(seqs, kv, group, n).permute(0, 3, 1, 2).reshape(seqs, n, c["heads"])[s["seq"], s["at"]]


def _plain_join(s):
    c = s["case"]
    parts, lses = [], []
    for x, l, rows in zip(s["parts"], s["lses"], s["rows"]):
        x = x.float()
        if rows is not None:
            there = rows >= 0
            x, l = x[rows.clamp(min=0).long()], torch.where(there[:, None], l[rows.clamp(min=0).long()], -math.inf)
        parts.append(x)
        lses.append(l)
    l = torch.stack(lses)
    m = l.amax(0)
    m = torch.where(m == -math.inf, 0.0, m)
    w = torch.exp(l - m)
    total = w.sum(0)
    o = sum(w[i, ..., None] * torch.where(w[i, ..., None] > 0, x, 0.0) for i, x in enumerate(parts))
    o = (o / torch.where(total > 0, total, 1.0)[..., None]).to(TYPES[c["dtype"]])
    return (o, m + torch.log(total)) if c["lse"] else o


_own = {"pages": _own_pages, "copy": _own_copy, "compact": _own_compact, "cross": _own_cross, "join": _own_join}
_plain = {"pages": _plain_pages, "copy": _plain_copy, "compact": _plain_compact, "cross": _plain_cross, "join": _plain_join}


# The definitions in 64 bits, or in whole numbers, one sequence after the other.

def _exact_pages(c, s):
    bs, blocks = c["block"], s["refs"].numel()
    old, lens, refs = s["table"].tolist(), s["lengths"].tolist(), s["kept"].tolist()
    upto, keep, width = s["upto"].tolist(), s["keep"].tolist(), s["table"].shape[1]
    table, lengths = [], []
    for p in s["parents"].tolist():
        table.append(list(old[p]) if 0 <= p < len(old) else [-1] * width)
        lengths.append(lens[p] if 0 <= p < len(old) else 0)
    for rows, sign in ((table, 1), (old, -1)):
        for row in rows:
            for p in row:
                if 0 <= p < blocks:
                    refs[p] += sign
    grows = [n < u <= width * bs for n, u in zip(lengths, upto)]
    ends = {}
    for b, n in enumerate(lengths):
        if grows[b] and n % bs and 0 <= table[b][n // bs] < blocks:
            ends.setdefault(table[b][n // bs], []).append(b)
    last = {v[-1] for p, v in ends.items() if len(v) > 1 and len(v) == refs[p]}
    free = [p for p in range(blocks) if refs[p] == 0]
    before, taken, now, src, dst = list(refs), 0, [], [], []
    for b, (n, u) in enumerate(zip(lengths, upto)):
        now.append(0)
        src.append(-1)
        dst.append(-1)
        if not grows[b]:
            now[b] = n if u <= n else 0
            continue
        places = []
        for j in range(n // bs, -(-u // bs)):
            p = table[b][j]
            valid = 0 <= p < blocks
            many = valid and before[p] > 1
            if j == n // bs and n % bs:
                if many and b not in last:
                    places.append(j)
            elif many or not valid:
                places.append(j)
        begin, taken = taken, taken + len(places)
        if taken > len(free) and (places or b in last):
            continue
        for i, j in enumerate(places):
            p, q = table[b][j], free[begin + i]
            if 0 <= p < blocks:
                refs[p] -= 1
            refs[q] += 1
            table[b][j] = q
            if j == n // bs and n % bs:
                src[b], dst[b] = p, q
        now[b] = lengths[b] = u
    for b in range(len(table)):
        lengths[b] = min(lengths[b], max(0, keep[b]))
        for j in range(-(-lengths[b] // bs), width):
            p, table[b][j] = table[b][j], -1
            if 0 <= p < blocks:
                refs[p] -= 1
    return {"table": _ints(table), "lengths": _ints(lengths), "refs": _ints(refs), "now": _ints(now), "src": _ints(src),
            "dst": _ints(dst)}


def _doubles(p):
    s = p["scale"].double()
    return {"k": p["k"].double() * s[..., 0, None, None], "v": p["v"].double() * s[..., 1, None, None], "scale": s,
            "bound": p["bound"].double() * s[..., 0, None, None]}


def _exact_copy(c, s):
    if c["real"] * c["layers"] * c["kv_heads"] * c["dim"] * c["block"] > 1 << 30:
        return None
    to, got = _doubles(s["to"]), _doubles(s["from"])
    for p, q in zip(s["src"].tolist(), s["dst"].tolist()):
        if p >= 0:
            for name in to:
                to[name][:, q] = got[name][:, p]
    return to


def _scale64(a):
    return 2.0 ** max(LEAST, math.ceil(math.log2(a / 127.0))) if a > 0 else 2.0 ** LEAST


def _exact_compact(c, s):
    kv, dim, bs = c["kv_heads"], c["dim"], c["block"]
    if sum(_counts(c)) * kv > 1 << 21 or sum(-(-n // bs) for n in _counts(c)) * kv > 12000:
        return None
    out, table, into = _doubles(s["to"]), s["table"], s["into_table"].tolist()
    k, v, scale = s["from"]["k"][0], s["from"]["v"][0], s["from"]["scale"][0].double()
    sizes = out["scale"].cpu()
    for b, n in enumerate(_counts(c)):
        for h in range(kv):
            at = s["keep"][b, 0 if c["same"] else h, :n].long()
            ids, slot = table[b, at // bs].long(), at % bs
            x = [k[ids, h, slot].double() * scale[ids, h, 0, None], v[ids, h, :, slot].double() * scale[ids, h, 1, None]]
            top = [torch.stack([p.abs().amax() for p in y.split(bs)]).tolist() for y in x]
            for j in range(-(-n // bs)):
                p, part = into[b][j], slice(j * bs, min(n, (j + 1) * bs))
                for i, name in ((0, "k"), (1, "v")):
                    step = _scale64(top[i][j])
                    y = torch.round(x[i][part] / step) * step
                    full = torch.zeros((bs, dim), dtype=torch.float64, device="cuda")
                    full[:len(y)] = y
                    out[name][0, p, h] = full if i == 0 else full.T
                    sizes[0, p, h, i] = step
                    if i == 0:
                        out["bound"][0, p, h, 0], out["bound"][0, p, h, 1] = y.amax(0), y.amin(0)
    return {**out, "scale": sizes.cuda()}


def _exact_cross(c, s):
    lens, news = _lengths(c)
    group, bs = c["heads"] // c["kv_heads"], c["block"]
    scale, out, sums, at = s["scale"].double(), [], [], 0
    for b, (n, m) in enumerate(zip(lens, news)):
        q = s["q"][at:at + m].double()
        at += m
        o = torch.zeros_like(q)
        l = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        ids = s["table"][b, :-(-n // bs)].long()
        for h in range(c["kv_heads"] if n else 0):
            k = (s["k"][ids, h].double() * scale[ids, h, 0, None, None]).reshape(-1, c["dim"])[:n]
            v = (s["v"][ids, h].double() * scale[ids, h, 1, None, None]).transpose(1, 2).reshape(-1, c["dim"])[:n]
            for f in range(h * group, (h + 1) * group):
                logits = (q[:, f] @ k.T) / math.sqrt(c["dim"])
                l[:, f] = torch.logsumexp(logits, 1)
                o[:, f] = torch.softmax(logits, 1) @ v
        out.append(o)
        sums.append(l)
    return (torch.cat(out), torch.cat(sums)) if c["lse"] else torch.cat(out)


def _exact_join(c, s):
    shape = (c["parts"], c["tokens"], c["heads"])
    l = torch.full(shape, -math.inf, dtype=torch.float64, device="cuda")
    x = torch.zeros((*shape, c["dim"]), dtype=torch.float64, device="cuda")
    for i, rows in enumerate(s["rows"]):
        there = torch.arange(c["tokens"], device="cuda") if rows is None else torch.nonzero(rows >= 0)[:, 0]
        which = there if rows is None else rows[there].long()
        l[i, there], x[i, there] = s["lses"][i][which].double(), s["parts"][i][which].double()
    total = torch.logsumexp(l, 0)
    w = torch.exp(l - torch.where(torch.isinf(total), 0.0, total))
    o = (w[..., None] * x).sum(0)
    return (o, total) if c["lse"] else o


def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "copy": _exact_copy, "compact": _exact_compact, "cross": _exact_cross,
            "join": _exact_join}[case["op"]](case, s)
