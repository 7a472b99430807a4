"""The key-value cache operators (include/dance_kv.h, dance_amd/kv.py) against
their definitions in 64 bits on the CPU.

Codes, scales, bounds and selections have to be equal. Attention's tolerance is the sum of
its roundings: the output's type (unit roundoff u), the weights in f16 (2^-11 of
each weight times its value), and the logits, float32 sums of dim products. With
A = sum p |v| and G = scale * max sum |q k| a row may be off by
u |o| + (2^-11 + 2 d + 2^-18) A, its logarithm by d + 2^-20 (1 + |lse|), where
d = G (dim + 8) 2^-24."""
import math
import re
import subprocess

import numpy as np
import pytest
import torch

import dance_amd as D
from dance_amd import kv

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}  # least positive numbers


# ------------------------------------------------------------- definitions

def scale_of(a):
    """Least 2^e, e >= -100, with a <= 127 * 2^e."""
    e = -100
    while a > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def codes_of(x, s):
    x = np.where(np.isnan(x), 0.0, x)
    return np.clip(np.rint(x / s), -127, 127)


class Model:
    """The cache in numpy, with the operators' definitions."""

    def __init__(self, cache):
        self.k, self.v = cache.k.cpu().numpy().astype(np.float64), cache.v.cpu().numpy().astype(np.float64)
        self.scale, self.bound = cache.scale.cpu().numpy().astype(np.float64), cache.bound.cpu().numpy().astype(np.int64)
        self.blocks, self.heads, self.bs, self.dim = self.k.shape

    def has(self, p):
        return 0 <= p < self.blocks

    def append(self, k, v, table, lengths, offsets):
        for b, n in enumerate(lengths):
            rows = range(offsets[b], offsets[b + 1])
            pos = [n - len(rows) + i for i in range(len(rows))]
            for j in range(table.shape[1]):
                new = [(r, p - j * self.bs) for r, p in zip(rows, pos) if p >= 0 and p // self.bs == j]
                if not new or not self.has(table[b, j]):
                    continue
                ph, old = table[b, j], new[0][1]
                for h in range(self.heads):
                    for i, (x, store) in enumerate(((k, self.k[ph, h]), (v, self.v[ph, h].T))):
                        part = np.array([x[r, h] for r, _ in new])
                        a = np.abs(part)
                        s = scale_of(a[np.isfinite(a)].max(initial=0.0))
                        if old:
                            s = max(s, self.scale[ph, h, i])
                            store[:old] = np.rint(store[:old] * self.scale[ph, h, i] / s)
                        else:
                            store[:] = 0
                        store[old:old + len(new)] = codes_of(part, s)
                        self.scale[ph, h, i] = s
                    live = self.k[ph, h, :old + len(new)]
                    self.bound[ph, h] = live.max(0), live.min(0)

    def attend(self, q, ids, pos, logical, scale):
        """One row of one head over the blocks ids (physical) that stand at `logical`."""
        h, q = q
        keys, vals = [], []
        for p, lg in zip(ids, logical):
            t = min(self.bs, pos - lg * self.bs + 1)
            if t > 0 and self.has(p):
                keys.append(self.k[p, h, :t] * self.scale[p, h, 0])
                vals.append(self.v[p, h, :, :t].T * self.scale[p, h, 1])
        if not keys:
            return np.zeros(self.dim), -math.inf, np.zeros(self.dim), 0.0
        keys, vals = np.concatenate(keys), np.concatenate(vals)
        x = keys @ q * scale
        m = x.max()
        p = np.exp(x - m)
        lse = m + math.log(p.sum())
        p /= p.sum()
        return p @ vals, lse, p @ np.abs(vals), float((np.abs(keys) @ np.abs(q)).max() * abs(scale))

    def attention(self, q, table, lengths, offsets, scale, lists=None):
        t, heads, dim = q.shape
        group = heads // self.heads
        out = [np.zeros((t, heads, dim)), np.full((t, heads), -math.inf), np.zeros((t, heads, dim)), np.zeros((t, heads))]
        room = table.shape[1] * self.bs
        for b, n in enumerate(lengths):
            m = offsets[b + 1] - offsets[b]
            for i in range(m):
                r, pos = offsets[b] + i, min(n - m + i, room - 1)
                for f in range(heads):
                    h = f // group
                    if lists is None:
                        lg = list(range(max(0, pos // self.bs + 1)))
                    else:
                        lg = [x for x in lists[r, h] if 0 <= x < table.shape[1]]
                    for k, x in enumerate(self.attend((h, q[r, f]), [table[b, j] for j in lg], pos, lg, scale)):
                        out[k][r, f] = x
        return out

    def select(self, q, table, lengths, offsets, count, sink, recent):
        t, heads, dim = q.shape
        group = heads // self.heads
        out = np.full((t, self.heads, count), -1, np.int32)
        for b, n in enumerate(lengths):
            m = offsets[b + 1] - offsets[b]
            for i in range(m):
                r, pos = offsets[b] + i, min(n - m + i, table.shape[1] * self.bs - 1)
                seen = pos // self.bs + 1 if pos >= 0 else 0
                for h in range(self.heads):
                    rank = []
                    for j in range(seen):
                        p = table[b, j]
                        if not self.has(p):
                            continue
                        best = -math.inf
                        for f in range(h * group, (h + 1) * group):
                            a = np.abs(q[r, f])
                            s = scale_of(a[np.isfinite(a)].max(initial=0.0))
                            c = codes_of(q[r, f], s)
                            total = np.maximum(c * self.bound[p, h, 0], c * self.bound[p, h, 1]).sum()
                            # the score is held in float32: one rounding, where the scale is no power of two
                            best = max(best, float(np.float32(total * self.scale[p, h, 0])) * s)
                        if j < sink or j >= seen - recent:
                            best = math.inf
                        rank.append((-best, j))
                    got = sorted(j for _, j in sorted(rank)[:count])
                    out[r, h, :len(got)] = got
        return out


# -------------------------------------------------------------- inputs

def make(rng, heads, dim, bs, lens, holes=0, spare=3, pow2=True, device="cuda"):
    """A cache with random codes, its sequences' table (as numpy too); blocks of no sequence hold rubbish."""
    wide = max(1, max(-(-n // bs) for n in lens)) + 1
    need = sum(-(-n // bs) for n in lens)
    pool = need + spare
    ids = rng.permutation(pool)
    table, at = np.full((len(lens), wide), -1, np.int32), 0
    for b, n in enumerate(lens):
        w = -(-n // bs)
        table[b, :w] = ids[at:at + w]
        at += w
    k = rng.integers(-127, 128, (pool, heads, bs, dim), dtype=np.int8)
    v = rng.integers(-127, 128, (pool, heads, dim, bs), dtype=np.int8)
    scale = 2.0 ** rng.integers(-9, -4, (pool, heads, 2)) if pow2 else rng.uniform(0.005, 0.03, (pool, heads, 2))
    scale = scale.astype(np.float32)
    scale[ids[at:]] = np.nan
    bound = np.stack((k.max(2), k.min(2)), 2)
    for _ in range(holes):
        b = rng.integers(len(lens))
        if table[b].max() >= 0:
            table[b, rng.integers(max(1, -(-lens[b] // bs)))] = rng.choice([-1, -7, pool, 2 ** 31 - 1])
    t = [torch.from_numpy(np.ascontiguousarray(x)).to(device) for x in (k, v, scale, bound)]
    return kv.KVCache(*t), table


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def offsets_of(news):
    return np.concatenate(([0], np.cumsum(news))).astype(np.int32)


def numbers(t):
    return t.double().cpu().numpy()


def check_attention(model, got, lse, q, table, lens, off, scale, lists=None):
    o, l, absolute, g = model.attention(numbers(q), table, lens, off, scale, lists)
    d = g * (model.dim + 8) * 2.0 ** -24
    least = LEAST[q.dtype]  # subnormal values are those that the output's type has
    o = np.where(np.abs(o) < least / ROUND[q.dtype], np.rint(o / least) * least, o)
    tol = ROUND[q.dtype] * np.abs(o) + (2.0 ** -11 + 2 * d[..., None] + 2.0 ** -18) * absolute
    err = np.abs(numbers(got) - o)
    assert (err <= tol).all(), (float((err - tol).max()), np.unravel_index((err - tol).argmax(), err.shape))
    if lse is not None:
        lse = numbers(lse)
        seen = np.isfinite(l)
        assert (np.isneginf(lse) == ~seen).all()
        assert (np.abs(lse[seen] - l[seen]) <= (d + 2.0 ** -20 * (1 + np.abs(np.where(seen, l, 0))))[seen]).all()


F16, BF16 = torch.float16, torch.bfloat16

# kv heads, group, dim, block tokens, type, lengths, rows of each sequence (None: one, without offsets)
SHAPES = [
    (2, 4, 128, 64, BF16, [1, 63, 64, 65, 0, 700], None),
    (1, 1, 64, 16, F16, [15, 16, 17, 1, 129], None),
    (3, 7, 96, 32, BF16, [5, 200, 33], [5, 1, 3]),
    (2, 3, 192, 128, F16, [127, 128, 129, 300], [2, 0, 4, 7]),
    (1, 16, 256, 64, BF16, [64, 321], [1, 2]),
    (1, 17, 128, 32, F16, [90, 31], None),
    (2, 1, 128, 16, BF16, [70, 3, 250], [40, 5, 1]),
    (2, 5, 64, 128, F16, [513, 130], [130, 130]),
    (1, 12, 96, 64, BF16, [0, 2, 190], [2, 4, 20]),  # rows before the sequence's first token
    (8, 4, 128, 64, F16, [260], None),
]
IDS = [f"{s[0]}x{s[1]}-{s[2]}-{s[3]}-{str(s[4])[6:]}-{i}" for i, s in enumerate(SHAPES)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("holes", [0, 2])
def test_attention(shape, holes):
    heads, group, dim, bs, dt, lens, news = shape
    rng = np.random.default_rng(1)
    cache, table = make(rng, heads, dim, bs, lens, holes)
    off = offsets_of(news or [1] * len(lens))
    q = torch.from_numpy(rng.normal(size=(off[-1], heads * group, dim))).to(dt).cuda()
    got, lse = kv.attention(cache, q, dev(table), dev(np.int32(lens)), dev(off) if news else None, return_lse=True,
                            max_tokens=max(news) if news else None)
    check_attention(Model(cache), got, lse, q, table, lens, off, dim ** -0.5)


# many rows of a sequence: prompts, their chunks, with earlier tokens and without
PROMPTS = [
    (1, 4, 128, 64, BF16, [200, 333, 0, 64], [200, 70, 3, 64]),
    (2, 3, 96, 32, F16, [257, 31, 1], [257, 31, 1]),
    (1, 2, 192, 16, BF16, [150, 65], [130, 65]),
    (1, 1, 256, 128, F16, [129, 400], [129, 90]),
    (3, 1, 64, 16, BF16, [300, 20, 90], [100, 33, 90]),
    (1, 24, 128, 32, F16, [70, 9], [20, 12]),      # rows before the first token
    (1, 2, 64, 64, BF16, [5000, 4100], [40, 60]),  # few rows over many tokens: split
    (9, 2, 64, 32, BF16, [64, 130, 70], [64, 40, 70]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", PROMPTS, ids=[f"{s[0]}x{s[1]}-{s[2]}-{s[3]}-{str(s[4])[6:]}" for s in PROMPTS])
@pytest.mark.parametrize("holes,scale", [(0, None), (3, 0.3), (0, -0.1), (0, 0.0)])
def test_attention_of_prompts(shape, holes, scale):
    heads, group, dim, bs, dt, lens, news = shape
    rng = np.random.default_rng(17)
    cache, table = make(rng, heads, dim, bs, lens, holes, pow2=scale is None)
    off = offsets_of(news)
    q = torch.from_numpy(rng.normal(size=(off[-1], heads * group, dim))).to(dt).cuda()
    got, lse = kv.attention(cache, q, dev(table), dev(np.int32(lens)), dev(off), scale=scale, return_lse=True,
                            max_tokens=max(news))
    check_attention(Model(cache), got, lse, q, table, lens, off, dim ** -0.5 if scale is None else scale)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("pow2", [True, False])
def test_select_and_sparse_attention(shape, pow2):
    heads, group, dim, bs, dt, lens, news = shape
    rng = np.random.default_rng(2)
    cache, table = make(rng, heads, dim, bs, lens, 2, pow2=pow2)
    off = offsets_of(news or [1] * len(lens))
    q = torch.from_numpy(rng.normal(size=(off[-1], heads * group, dim))).to(dt).cuda()
    args = dev(table), dev(np.int32(lens))
    model = Model(cache)
    for count, sink, recent in ((1, 0, 0), (2, 0, 1), (3, 1, 1), (40, 1, 2)):
        got = kv.select(cache, q, *args, count, dev(off) if news else None, sink=sink, recent=recent)
        assert (got.cpu().numpy() == model.select(numbers(q), table, lens, off, count, sink, recent)).all()
    # lists in any order, with entries that are nowhere
    lists = np.full((off[-1], heads, 5), -1, np.int32)
    for x in lists.reshape(-1, 5):
        x[:] = rng.permutation(np.concatenate((np.arange(table.shape[1]), [-1, -9, 1 << 30, table.shape[1] + 3, 70])))[:5]
    for x in (lists, np.ascontiguousarray(lists[:, :, :1])):
        o, lse = kv.sparse_attention(cache, q, dev(x), *args, dev(off) if news else None, scale=0.2, return_lse=True)
        check_attention(model, o, lse, q, table, lens, off, 0.2, x)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_append(shape):
    """Prompts, then single tokens, some of which make their block grow."""
    heads, _, dim, bs, dt, lens, news = shape
    rng = np.random.default_rng(3)
    lens = np.maximum(lens, 1)
    cache, table = make(rng, heads, dim, bs, [n + 3 for n in lens], 1)
    model = Model(cache)
    for step in range(4):
        n = np.int32(lens if step == 0 else np.ones(len(lens)))
        off, now = offsets_of(n), np.int32(lens + step)
        x = rng.normal(size=(2, off[-1], heads, dim)) * (1.0, 0.4, 5.0, 40.0)[step] * rng.uniform(0.01, 1, (2, 1, 1, dim))
        k, v = (torch.from_numpy(y).to(dt).cuda() for y in x)
        kv.append(cache, k, v, dev(table), dev(now), dev(off) if step == 0 else None, max_tokens=int(n.max()))
        model.append(numbers(k), numbers(v), table, now, off)
        written = np.unique(table[(table >= 0) & (table < cache.blocks)])
        assert (numbers(cache.scale)[written] == model.scale[written]).all()
        assert (numbers(cache.k) == model.k).all() and (numbers(cache.v) == model.v).all()
        assert (cache.bound.cpu().numpy() == model.bound).all()


@pytest.mark.gpu
def test_append_in_parts_of_any_size():
    """A prompt that comes in parts, from the middle of a block to the middle of another."""
    rng = np.random.default_rng(4)
    cache, table = make(rng, 2, 64, 16, [200])
    model, n = Model(cache), 0
    for part in (5, 11, 3, 40, 1, 30, 17, 93):
        n += part
        k, v = (torch.from_numpy(rng.normal(size=(part, 2, 64)) * rng.choice([0.1, 1, 3])).to(BF16).cuda() for _ in range(2))
        off = np.int32([0, part])
        kv.append(cache, k, v, dev(table), dev(np.int32([n])), dev(off))
        model.append(numbers(k), numbers(v), table, [n], off)
    assert (numbers(cache.k) == model.k).all() and (numbers(cache.v) == model.v).all()
    ids = table[0, :13]
    assert (numbers(cache.scale)[ids] == model.scale[ids]).all() and (cache.bound.cpu().numpy() == model.bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_append_of_extreme_values(dt):
    rng = np.random.default_rng(5)
    cache, table = make(rng, 1, 64, 16, [16] * 7)
    x = rng.normal(size=(2, 7 * 16, 1, 64))
    x[:, 0:16] = 0.0                                  # a block of zeros takes the least scale
    x[:, 16:32] *= 1e-30 if dt == BF16 else 6e-8      # subnormal in float16
    x[:, 32, 0, :3] = np.inf, -np.inf, np.nan         # infinities saturate, NaN is 0, neither sets the scale
    x[:, 48:64] = np.nan
    x[:, 64] = float(torch.finfo(dt).max)
    x[:, 80:96] = 127 * 2.0 ** -3                     # exactly the largest value of a scale
    x[:, 96:112] = 127.5 * 2.0 ** -3
    k, v = (torch.from_numpy(y).to(dt).cuda() for y in x)
    off, lens = offsets_of([16] * 7), np.int32([16] * 7)
    model = Model(cache)
    kv.append(cache, k, v, dev(table), dev(lens), dev(off))
    with np.errstate(invalid="ignore"):
        model.append(numbers(k), numbers(v), table, lens, off)
    ids = table[:, 0]
    assert (numbers(cache.scale)[ids] == model.scale[ids]).all()
    assert (numbers(cache.k) == model.k).all() and (numbers(cache.v) == model.v).all()


@pytest.mark.gpu
def test_append_divides_by_scales_that_are_no_powers_of_two():
    """A cache that another program filled: its scales stay while they hold the new values."""
    rng = np.random.default_rng(6)
    cache, table = make(rng, 2, 128, 32, [40, 90], pow2=False)
    model = Model(cache)
    k, v = (torch.from_numpy(rng.normal(size=(2, 2, 128)) * 0.1).to(BF16).cuda() for _ in range(2))
    kv.append(cache, k, v, dev(table), dev(np.int32([40, 90])))
    ids = [table[0, 1], table[1, 2]]
    assert (numbers(cache.scale)[ids] == model.scale[ids]).all()  # held: 127 x 0.005 is above 0.1 x 5 sigma
    for i, (x, store) in enumerate(((k, cache.k), (v, cache.v.transpose(2, 3)))):
        for b, (p, slot) in enumerate(((ids[0], 7), (ids[1], 25))):
            for h in range(2):
                s = np.float32(model.scale[p, h, i])
                want = np.clip(np.rint(numbers(x)[b, h].astype(np.float32) / s), -127, 127)
                assert (store[p, h, slot].cpu().numpy() == want).all()


@pytest.mark.gpu
def test_values_hidden_or_behind_the_end_change_nothing():
    """Rubbish in blocks of no sequence, in slots behind the last token and in later tokens of a prompt."""
    rng = np.random.default_rng(7)
    lens, news = [100, 37], [60, 37]
    cache, table = make(rng, 2, 128, 32, lens)
    off = offsets_of(news)
    q = torch.from_numpy(rng.normal(size=(97, 4, 128))).to(BF16).cuda()
    args = dev(table), dev(np.int32(lens)), dev(off)
    want = kv.attention(cache, q, *args, max_tokens=60)
    rows = [off[0] + 10, off[1] + 5]  # positions 50 and 5
    for p in range(cache.blocks):
        where = np.argwhere(table == p)
        start = 51 if len(where) and where[0][0] == 0 else 6
        first = where[0][1] * 32 if len(where) else 1 << 30
        for t in range(32):
            if first + t >= start:
                cache.k[p, :, t] = 127
                cache.v[p, :, :, t] = -127
    got = kv.attention(cache, q, *args, max_tokens=60)
    assert torch.equal(got[rows], want[rows])
    assert not torch.equal(got, want)


@pytest.mark.gpu
def test_peaked_flat_and_infinite_logits():
    rng = np.random.default_rng(8)
    lens = [500, 500, 500, 500]
    cache, table = make(rng, 1, 128, 64, lens)
    q = rng.normal(size=(4, 2, 128))
    q[0] *= 200.0   # all weight on a token
    q[1] = 0.0      # equal weights
    q[2] *= 1e-4
    q = torch.from_numpy(q).to(BF16).cuda()
    got, lse = kv.attention(cache, q, dev(table), dev(np.int32(lens)), return_lse=True)
    check_attention(Model(cache), got, lse, q, table, lens, offsets_of([1] * 4), 128 ** -0.5)
    q[3, 1, 5] = math.nan
    bad = kv.attention(cache, q, dev(table), dev(np.int32(lens)))
    assert torch.equal(bad[:3], got[:3]) and torch.equal(bad[3, 0], got[3, 0]) and bad[3, 1].isnan().all()


@pytest.mark.gpu
def test_value_scales_of_any_ratio():
    """Blocks whose values are zero or tiny count in the softmax like others."""
    rng = np.random.default_rng(9)
    lens = [640]
    cache, table = make(rng, 1, 64, 64, lens)
    cache.scale[..., 1] = torch.from_numpy(np.float32([2.0 ** e for e in rng.integers(-60, 3, cache.blocks)]))[:, None].cuda()
    cache.v[int(table[0, 3])] = 0
    cache.scale[int(table[0, 3]), 0, 1] = 0.0
    q = torch.from_numpy(rng.normal(size=(1, 4, 64))).to(F16).cuda()
    got, lse = kv.attention(cache, q, dev(table), dev(np.int32(lens)), return_lse=True)
    check_attention(Model(cache), got, lse, q, table, lens, [0, 1], 64 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("news", [[8, 3], [90, 70]])
def test_rows_that_see_nothing_give_zeros_whatever_their_queries(dt, news):
    """Rows before the first token, over holes alone, or with empty lists, beside rows that see tokens."""
    rng = np.random.default_rng(18)
    lens = [3, 75]
    cache, table = make(rng, 2, 128, 16, lens)
    table[1] = -1
    off = offsets_of(news)
    q = torch.from_numpy(rng.normal(size=(off[-1], 4, 128))).to(dt).cuda()
    blind = torch.tensor([i < news[0] - 3 or i >= news[0] for i in range(off[-1])], device="cuda")
    args = dev(table), dev(np.int32(lens)), dev(off)
    lists = np.tile(np.int32([0, -1, 4, 1]), (off[-1], 2, 1))
    lists[news[0] - 1] = -1
    unlisted = blind.clone()
    unlisted[news[0] - 1] = True

    def both(x):
        return [kv.attention(cache, x, *args, max_tokens=max(news), return_lse=True),
                kv.sparse_attention(cache, x, dev(lists), *args, max_tokens=max(news), return_lse=True)]
    want = both(q)
    for value in (math.nan, math.inf, -math.inf):
        for hidden, i in ((blind, 0), (unlisted, 1)):
            bad = q.clone()
            bad[hidden] = value
            bad[hidden, :, 5] = 1.0
            o, lse = both(bad)[i]
            assert torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])
            assert (o[hidden] == 0).all() and torch.isneginf(lse[hidden]).all()


@pytest.mark.gpu
def test_large_keys_and_small_queries():
    """Powers of two that the keys have and the queries lack change nothing, far beyond the logits' range."""
    rng = np.random.default_rng(19)
    lens, news = [200, 90], [3, 70]
    cache, table = make(rng, 1, 128, 32, lens)
    q = torch.from_numpy(rng.normal(size=(73, 2, 128))).to(BF16).cuda()
    args = dev(table), dev(np.int32(lens))

    def with_keys(e):
        scale = cache.scale.clone()
        scale[..., 0] *= 2.0 ** e
        return kv.KVCache(cache.k, cache.v, scale, cache.bound)
    for x, off in ((q[:2], None), (q, dev(offsets_of(news)))):
        want = kv.attention(cache, x, *args, off, scale=0.1, return_lse=True)
        got = kv.attention(with_keys(112), x * 2.0 ** -100, *args, off, scale=0.1 * 2.0 ** -12, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        chosen = kv.select(with_keys(28), x, *args, 2, off)
        assert torch.equal(chosen, kv.select(with_keys(118), x * 2.0 ** -90, *args, 2, off))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_rows_with_strides_and_odd_addresses(dt):
    """Queries, keys and values as slices of one projection's rows, aligned and not."""
    rng = np.random.default_rng(10)
    lens = [70, 33, 5]
    cache, table = make(rng, 2, 96, 32, lens)
    args = dev(table), dev(np.int32(lens))
    base = torch.from_numpy(rng.normal(size=(3, 8 * 97 + 1))).to(dt).cuda()
    for x in (base[:, 1:].view(3, 8, 97)[:, :, 1:], base[:, :8 * 96].view(3, 8, 96)):
        q, k, v = x[:, :4], x[:, 4:6], x[:, 6:8]
        assert torch.equal(kv.attention(cache, q, *args), kv.attention(cache, q.contiguous(), *args))
        assert torch.equal(kv.select(cache, q, *args, 2), kv.select(cache, q.contiguous(), *args, 2))
        other = kv.KVCache(cache.k.clone(), cache.v.clone(), cache.scale.clone(), cache.bound.clone())
        kv.append(other, k.contiguous(), v.contiguous(), *args)
        kv.append(cache, k, v, *args)
        assert torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v) and torch.equal(cache.bound, other.bound)
    # the heads of all tokens together
    q = base[:, :8 * 96].view(3, 8, 96)[:, :4].transpose(0, 1).contiguous().transpose(0, 1)
    assert q.stride(0) < q.stride(1)
    assert torch.equal(kv.attention(cache, q, *args), kv.attention(cache, q.contiguous(), *args))


@pytest.mark.gpu
def test_long_context_is_split_and_joined():
    rng = np.random.default_rng(11)
    lens = [9001, 1, 4097]
    cache, table = make(rng, 1, 64, 64, lens)
    q = torch.from_numpy(rng.normal(size=(3, 2, 64)) * 3).to(F16).cuda()
    args = dev(table), dev(np.int32(lens))
    got, lse = kv.attention(cache, q, *args, return_lse=True)
    check_attention(Model(cache), got, lse, q, table, lens, offsets_of([1] * 3), 64 ** -0.5)
    again = kv.attention(cache, q, *args)
    assert torch.equal(got, again)
    hinted = kv.attention(cache, q, *args, max_length=9001)
    assert (hinted.float() - got.float()).abs().max() < 2.0 ** -8
    lists = np.stack([np.pad(rng.permutation(-(-n // 64))[:100], (0, 100), constant_values=-1)[:100] for n in lens])
    lists = np.int32(lists)[:, None]
    o, lse = kv.sparse_attention(cache, q, dev(lists), *args, return_lse=True)
    check_attention(Model(cache), o, lse, q, table, lens, offsets_of([1] * 3), 64 ** -0.5, lists)


@pytest.mark.gpu
def test_select_over_many_blocks_with_equal_scores():
    """Every fourth block has the same bounds: equal scores go to the lower block."""
    rng = np.random.default_rng(12)
    lens = [16 * 3000]
    cache, table = make(rng, 2, 64, 16, lens)
    cache.bound[:] = cache.bound[torch.arange(cache.blocks, device="cuda") % 4]
    cache.scale[..., 0] = 0.125
    q = torch.from_numpy(rng.normal(size=(1, 4, 64))).to(BF16).cuda()
    model = Model(cache)
    for count in (5, 700, 1200, 2999, 3000, 3500):
        got = kv.select(cache, q, dev(table), dev(np.int32(lens)), count, sink=1, recent=1)
        assert (got.cpu().numpy() == model.select(numbers(q), table, lens, [0, 1], count, 1, 1)).all()


@pytest.mark.gpu
def test_selected_bound_holds_for_every_token():
    """The score of a block is no less than any token's product with the rounded query."""
    rng = np.random.default_rng(13)
    cache, table = make(rng, 1, 128, 32, [32 * 40])
    q = torch.from_numpy(rng.normal(size=(1, 1, 128))).to(BF16).cuda()
    x = numbers(q)[0, 0]
    s = scale_of(np.abs(x).max())
    c = np.rint(x / s) * s
    model = Model(cache)
    keys = model.k[table[0, :40], 0] * model.scale[table[0, :40], 0, 0][:, None, None]
    best = (keys @ c).max(1)
    bound = np.maximum(c * model.bound[table[0, :40], 0, 0], c * model.bound[table[0, :40], 0, 1]).sum(1) * model.scale[table[0, :40], 0, 0]
    assert (bound >= best).all()
    got = kv.select(cache, q, dev(table), dev(np.int32([32 * 40])), 8).cpu().numpy()[0, 0]
    assert set(got) == set(np.argsort(-bound, kind="stable")[:8])


@pytest.mark.gpu
def test_cache_beyond_32_bit_offsets():
    """Blocks whose codes lie more than 2^32 bytes into the arrays."""
    heads, bs, dim = 8, 128, 256
    blocks = (1 << 32) // (heads * bs * dim) + 40
    cache = kv.KVCache.empty(blocks, heads, dim, bs)
    rng = np.random.default_rng(14)
    small, _ = make(rng, heads, dim, bs, [300])
    table = np.int32([[blocks - 1, 3, blocks - 30]])
    near = np.int32([[0, 1, 2]])
    k, v = (torch.from_numpy(rng.normal(size=(300, heads, dim))).to(BF16).cuda() for _ in range(2))
    q = torch.from_numpy(rng.normal(size=(1, heads * 2, dim))).to(BF16).cuda()
    n, off = dev(np.int32([300])), dev(np.int32([0, 300]))
    got = []
    for c, t in ((cache, dev(table)), (small, dev(near))):
        kv.append(c, k, v, t, n, off)
        got.append((kv.attention(c, q, t, n), kv.select(c, q, t, n, 2), kv.sparse_attention(
            c, q, dev(np.tile(np.int32([0, 2]), (1, heads, 1))), t, n)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_graph_of_a_step_replays():
    """append, select and both attentions in a graph, replayed as the sequences grow."""
    rng = np.random.default_rng(15)
    lens = [130, 64]
    cache, table = make(rng, 2, 128, 32, [n + 40 for n in lens])
    eager = kv.KVCache(cache.k.clone(), cache.v.clone(), cache.scale.clone(), cache.bound.clone())
    t, n = dev(table), dev(np.int32(lens))
    x = torch.zeros((2, 12, 128), dtype=BF16, device="cuda")

    def step(c):
        kv.append(c, x[:, 8:10], x[:, 10:], t, n)
        chosen = kv.select(c, x[:, :8], t, n, 3, recent=1)
        return chosen, kv.sparse_attention(c, x[:, :8], chosen, t, n), kv.attention(c, x[:, :8], t, n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv.attention(eager, x[:, :8], t, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache)
    for i in range(5):
        n += 1
        x.copy_(torch.from_numpy(rng.normal(size=(2, 12, 128))))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)


@pytest.mark.gpu
def test_calls_run_on_the_current_stream():
    rng = np.random.default_rng(16)
    lens = [3000, 20]
    cache, table = make(rng, 2, 128, 64, lens)
    t, n = dev(table), dev(np.int32(lens))
    q = torch.from_numpy(rng.normal(size=(2, 8, 128))).to(BF16).cuda()
    want = kv.attention(cache, q, t, n)
    other = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-4
        other.copy_(q)  # behind the products: a call on another stream would read zeros
        got = kv.attention(cache, other, t, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_no_rows():
    cache = kv.KVCache.empty(2, 1, 64, 16)
    t, n, off = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((1, 2), (1,), (2,)))
    q = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    assert kv.attention(cache, q, t, n, off).shape == (0, 2, 64)
    assert kv.select(cache, q, t, n, 3, off).shape == (0, 1, 3)
    kv.append(cache, q[:, :1], q[:, :1], t, n, off)


# ------------------------------------------------------------- refusals

@pytest.mark.gpu
def test_refusals():
    cache = kv.KVCache.empty(4, 2, 64, 16)
    t, n = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    q = torch.zeros((3, 4, 64), dtype=BF16, device="cuda")
    k = q[:, :2]
    for exc, call in [
            (TypeError, lambda: kv.attention(cache, q.float(), t, n)),
            (ValueError, lambda: kv.attention(cache, q[:, :3], t, n)),
            (ValueError, lambda: kv.attention(cache, q[:, :0], t, n)),
            (ValueError, lambda: kv.attention(cache, q[:2], t, n)),
            (ValueError, lambda: kv.attention(cache, q.transpose(1, 2), t, n)),
            (ValueError, lambda: kv.attention(cache, q[..., :32], t, n)),
            (ValueError, lambda: kv.attention(cache, q.cpu(), t, n)),
            (TypeError, lambda: kv.attention(cache, q, t.long(), n)),
            (ValueError, lambda: kv.attention(cache, q, t, n[:2])),
            (ValueError, lambda: kv.attention(cache, q, t.t(), n)),
            (ValueError, lambda: kv.attention(cache, q, t, n, off[:3])),
            (ValueError, lambda: kv.attention(cache, q, t, n, off, max_tokens=0)),
            (ValueError, lambda: kv.attention(cache, q, t, n, max_length=0)),
            (ValueError, lambda: kv.attention(cache, q, t, n, out=q[:2])),
            (RuntimeError, lambda: kv.attention(cache, q, t, n, scale=math.nan)),
            (ValueError, lambda: kv.append(cache, q, q, t, n)),
            (ValueError, lambda: kv.append(cache, k, k[:2], t, n)),
            (ValueError, lambda: kv.append(cache, k, k.half(), t, n)),
            (ValueError, lambda: kv.select(cache, q, t, n, 0)),
            (ValueError, lambda: kv.select(cache, q, t, n, 2, sink=1, recent=2)),
            (ValueError, lambda: kv.sparse_attention(cache, q, t, t, n)),
            (TypeError, lambda: kv.sparse_attention(cache, q, torch.zeros((3, 2, 1), device="cuda"), t, n)),
            (ValueError, lambda: kv.sparse_attention(cache, q, torch.zeros((3, 1, 1), dtype=torch.int32, device="cuda"), t, n))]:
        with pytest.raises(exc):
            call()


def test_cache_refuses_arrays_that_do_not_fit():
    def arrays(blocks=3, heads=2, bs=16, dim=64):
        return [torch.zeros((blocks, heads, bs, dim), dtype=torch.int8), torch.zeros((blocks, heads, dim, bs), dtype=torch.int8),
                torch.zeros((blocks, heads, 2)), torch.zeros((blocks, heads, 2, dim), dtype=torch.int8)]
    with pytest.raises(ValueError, match="GPU"):
        kv.KVCache(*arrays())
    for bad in ({"bs": 24}, {"dim": 80}):
        with pytest.raises(ValueError, match="dim"):
            kv.KVCache(*arrays(**bad))
    for i in range(4):
        a = arrays()
        a[i] = a[i].to(torch.int16)
        with pytest.raises(TypeError):
            kv.KVCache(*a)
        a = arrays()
        a[i] = a[i][:2].clone() if i else a[i].transpose(0, 1)
        with pytest.raises(ValueError):
            kv.KVCache(*a)


def fake(**change):
    """Arguments whose pointers are never followed: every call with them is refused on the host."""
    c = dict(k=1 << 20, v=1 << 20, scale=1 << 20, bound=1 << 20, blocks=4, kv_heads=2, dim=64, block_tokens=16)
    b = dict(table=1 << 20, lengths=1 << 20, offsets=1 << 20, seqs=2, tokens=5, table_width=3, max_tokens=5, max_length=0)
    r = dict(data=1 << 20, token_stride=256, head_stride=64, heads=4, dtype=3)
    for key, x in change.items():
        for d in (c, b, r):
            if key in d:
                d[key] = x
    return kv.DanceKvCache(**c), kv.DanceKvBatch(**b), kv.DanceKvRows(**r)


REFUSED = [{"k": None}, {"bound": 1 << 20 | 4}, {"blocks": 0}, {"kv_heads": 0}, {"kv_heads": 3}, {"dim": 100},
           {"block_tokens": 48}, {"table": None}, {"lengths": None}, {"offsets": None}, {"seqs": 0}, {"table_width": 0},
           {"table_width": 1 << 28}, {"max_tokens": 0}, {"max_tokens": 6}, {"data": None}, {"data": 1 << 20 | 1},
           {"heads": 0}, {"dtype": 0}]


@pytest.mark.parametrize("change", REFUSED, ids=[str(x) for x in REFUSED])
def test_entries_refuse_before_any_device_work(change, capfd):
    L = kv._bind()
    c, b, r = fake(**change)
    big = 1 << 40
    assert L.dance_kv_attention(c, b, r, 1.0, 1 << 20, None, 1 << 20, big, None) == -1
    assert L.dance_kv_sparse_attention(c, b, r, 1 << 20, 2, 1.0, 1 << 20, None, 1 << 20, big, None) == -1
    assert L.dance_kv_select(c, b, r, 2, 0, 0, 1 << 20, 1 << 20, big, None) == -1
    if "heads" not in change:
        r.heads = 2
        c.kv_heads = change.get("kv_heads", 2)
        if "kv_heads" not in change or change["kv_heads"] != 2:
            assert L.dance_kv_append(c, b, r, r, None) == -1
    assert "dance_kv" in capfd.readouterr().err


def test_entries_refuse_what_else_is_missing(capfd):
    L = kv._bind()
    c, b, r = fake()
    assert L.dance_kv_attention(None, b, r, 1.0, 1 << 20, None, None, 0, None) == -1
    assert L.dance_kv_attention(c, None, r, 1.0, 1 << 20, None, None, 0, None) == -1
    assert L.dance_kv_attention(c, b, None, 1.0, 1 << 20, None, None, 0, None) == -1
    assert L.dance_kv_attention(c, b, r, 1.0, None, None, None, 0, None) == -1
    assert L.dance_kv_attention(c, b, r, math.inf, 1 << 20, None, None, 0, None) == -1
    assert L.dance_kv_append(c, b, r, r, None) == -1  # four heads of two
    r.heads = 2
    other = kv.DanceKvRows(r.data, 256, 64, 2, 2)
    assert L.dance_kv_append(c, b, r, other, None) == -1  # two types
    assert L.dance_kv_select(c, b, r, 0, 0, 0, 1 << 20, 1 << 20, 1 << 40, None) == -1
    assert L.dance_kv_select(c, b, r, 2, 1, 2, 1 << 20, 1 << 20, 1 << 40, None) == -1
    assert L.dance_kv_select(c, b, r, 2, 0, 0, None, 1 << 20, 1 << 40, None) == -1
    assert L.dance_kv_sparse_attention(c, b, r, None, 2, 1.0, 1 << 20, None, None, 0, None) == -1
    assert L.dance_kv_sparse_attention(c, b, r, 1 << 20, 0, 1.0, 1 << 20, None, None, 0, None) == -1
    # a workspace that is missing, too small or at an odd address
    b = fake(seqs=1, table_width=5000, tokens=1, max_tokens=1)[1]
    need = L.dance_kv_attention_work(c, b, 2)
    assert need > 0 and L.dance_kv_attention_work(c, b, 3) == 0
    for at, size in ((None, need), (1 << 20, need - 1), (1 << 20 | 8, need)):
        assert L.dance_kv_attention(c, b, r, 1.0, 1 << 20, None, at, size, None) == -1
    need = L.dance_kv_select_work(c, b, 2, 4)
    for at, size in ((None, need), (1 << 20, need - 1), (1 << 20 | 8, need)):
        assert need > 0 and L.dance_kv_select(c, b, r, 4, 0, 0, 1 << 20, at, size, None) == -1


def test_workspaces_of_lists_that_the_call_refuses():
    L = kv._bind()
    c, b, _ = fake(kv_heads=8, seqs=64, tokens=64, max_tokens=1, offsets=None)
    assert L.dance_kv_sparse_attention_work(c, b, 32, 1 << 20) > 0
    assert L.dance_kv_sparse_attention_work(c, b, 32, 0) == 0  # 512 units: more than one launch rule's 256
    assert L.dance_kv_sparse_attention_work(c, b, 32, 1 << 27) == 0


def test_a_longest_length_beyond_the_table_counts_as_the_table():
    L = kv._bind()
    for longest in (0, 5000 * 16, 1 << 40, (1 << 64) - 1):
        c, b, _ = fake(seqs=1, tokens=1, max_tokens=1, offsets=None, table_width=5000, max_length=longest)
        assert [L.dance_kv_attention_work(c, b, 4), L.dance_kv_select_work(c, b, 4, 8)] == [4 * 79 * 66 * 4, 2 * 5000 * 4]
    c, b, _ = fake(seqs=200, tokens=200, max_tokens=1, offsets=None, table_width=5000, max_length=(1 << 64) - 1)
    assert L.dance_kv_attention_work(c, b, 4) == 200 * 4 * 3 * 66 * 4  # 400 units: not one workgroup each


def test_library_exports_every_declared_entry():
    text = open(D.HERE + "/../include/dance_kv.h").read()
    names = set(re.findall(r"\b(dance_kv_\w+)\(const", text))
    assert len(names) == 7
    out = subprocess.run(["nm", "-D", "--defined-only", D.LIB_PATH], capture_output=True, text=True).stdout
    assert {n for n in names if f" T {n}\n" in out} == names


@pytest.mark.gpu
def test_example_of_a_decoding_loop():
    """The operators together: the selected blocks hold more of the weight than as many of the
    newest, and all blocks hold all of it."""
    import os
    import sys
    sys.path.insert(0, os.path.join(D.HERE, "..", "examples"))
    try:
        import kv_retrieval
    finally:
        sys.path.pop(0)
    some = kv_retrieval.run(seqs=3, prompt=9000, steps=4, count=24, quiet=True)
    assert all(s["newest"] < s["mass"] <= 1 + 2.0 ** -10 for s in some)
    every = kv_retrieval.run(seqs=2, prompt=3000, steps=2, count=64, quiet=True)
    assert all(abs(s["mass"] - 1) < 2.0 ** -10 and s["apart"] < 2.0 ** -7 for s in every)
