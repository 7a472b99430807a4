"""The key-value cache operators in calls that reach each of their kernels, also at small and odd
sizes: a wide table makes a call large for the launch rules, whatever its sequences hold. Every test
names the kernels that it means and asks torch's profiler which ran. Definitions: test_kv.py.

Attention's tolerance is the one of test_kv.py and what two formats add to it: an output is off by up to half the
least number of its type; a weight in f16 by 2^-11 of itself or 2^-25, where the largest weight times its
value's scale stands at 2^13 or more. So with the softmax's weights w, codes c and scales y, by
2^-38 max(w y) sum |c|."""
import re

import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, F16, LEAST, ROUND, Model, codes_of, dev, numbers, offsets_of, scale_of

pytestmark = pytest.mark.gpu


def launched(call):
    """The call's result and the library's kernels that it launched, as k_name<arguments>."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        out = call()
        torch.cuda.synchronize()
    names = " ".join(e.key for e in p.key_averages())
    return out, {re.sub(r"(\d)u\b", r"\1", n) for n in re.findall(r"\(anonymous namespace\)::(k_\w+(?:<[^>]*>)?)\(", names)}


@pytest.fixture(scope="module", autouse=True)
def kernels_have_names():
    cache = kv.KVCache.empty(1, 1, 64, 16)
    q, n = torch.zeros((1, 1, 64), dtype=BF16, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    if launched(lambda: kv.attention(cache, q, n[:, None] - 1, n))[1] != {"k_step<64, true, false, true, 8>"}:
        pytest.skip("torch's profiler does not name the kernels here")


def flag(x):
    return "true" if x else "false"


class Large(Model):
    """The same definitions for many rows and blocks: a product for each sequence and kv head, on the GPU in 64 bits."""

    def attention(self, q, table, lengths, offsets, scale, lists=None):
        t, heads, dim = q.shape
        group, wide = heads // self.heads, table.shape[1]
        out = [np.zeros((t, heads, dim)), np.full((t, heads), -np.inf), np.zeros((t, heads, dim)), np.zeros((t, heads)),
               np.zeros((t, heads, dim))]
        for b, n in enumerate(lengths):
            r0, m = offsets[b], offsets[b + 1] - offsets[b]
            used = min(wide, max(1, -(-n // self.bs)))
            ids = table[b, :used]
            live = (ids >= 0) & (ids < self.blocks)
            ids = np.where(live, ids, 0)
            pos = np.minimum(n - m + np.arange(m), wide * self.bs - 1)
            seen = (np.arange(used * self.bs) <= pos[:, None]) & np.repeat(live, self.bs)
            for h in range(self.heads if m else 0):
                keys = dev(self.k[ids, h] * self.scale[ids, h, 0, None, None]).view(-1, dim)
                codes = dev(self.v[ids, h].transpose(0, 2, 1)).reshape(-1, dim)
                y = dev(np.repeat(self.scale[ids, h, 1], self.bs))
                vals = codes * y[:, None]
                shown = seen
                if lists is not None:
                    listed = np.zeros((m, used + 1), bool)
                    at = lists[r0:r0 + m, h]
                    np.put_along_axis(listed, np.where((at >= 0) & (at < used), at, used), True, 1)
                    shown = seen & np.repeat(listed[:, :used], self.bs, 1)
                f = slice(h * group, (h + 1) * group)
                x = dev(q[r0:r0 + m, f]).reshape(-1, dim)
                hidden = ~dev(shown).repeat_interleave(group, 0)
                logits = (x @ keys.t().contiguous() * scale).masked_fill_(hidden, -np.inf)
                lse = torch.logsumexp(logits, 1)
                p = torch.exp(logits - torch.where(lse == -np.inf, 0.0, lse)[:, None])
                g = (x.abs() @ keys.abs().t().contiguous() * abs(scale)).masked_fill_(hidden, 0.0).amax(1)
                least = (p * y).amax(1, keepdim=True) * ((~hidden).double() @ codes.abs())
                for o, z, tail in zip(out, (p @ vals, lse, p @ vals.abs(), g, least), ((dim,), (), (dim,), (), (dim,))):
                    o[r0:r0 + m, f] = z.view(m, group, *tail).cpu().numpy()
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
                ids = table[b, :seen]
                live = (ids >= 0) & (ids < self.blocks)
                j = np.arange(seen)
                for h in range(self.heads):
                    best = np.full(self.blocks, -np.inf)
                    for x in q[r, h * group:(h + 1) * group]:
                        s = scale_of(np.abs(x).max(initial=0.0))
                        c = codes_of(x, s)
                        total = self.bound[:, h, 0] @ np.maximum(c, 0) + self.bound[:, h, 1] @ np.minimum(c, 0)
                        best = np.maximum(best, np.float32(total * self.scale[:, h, 0]).astype(np.float64) * s)
                    score = np.where(live, best[np.where(live, ids, 0)], -np.inf)
                    score = np.where(live & ((j < sink) | (j >= seen - recent)), np.inf, score)
                    order = np.lexsort((j, -score))
                    got = np.sort(order[score[order] > -np.inf][:count])
                    out[r, h, :len(got)] = got
        return out


def check(model, got, lse, q, table, lens, off, scale, lists=None):
    o, l, absolute, g, small = model.attention(numbers(q), table, lens, off, scale, lists)
    d = g * (model.dim + 8) * 2.0 ** -24
    tol = (ROUND[q.dtype] * np.abs(o) + LEAST[q.dtype] / 2 + (2.0 ** -11 + 2 * d[..., None] + 2.0 ** -18) * absolute
           + 2.0 ** -38 * small)
    err = np.abs(numbers(got) - o)
    assert (err <= tol).all(), (float((err - tol).max()), np.unravel_index((err - tol).argmax(), err.shape))
    lse, seen = numbers(lse), np.isfinite(l)
    assert (np.isneginf(lse) == ~seen).all()
    assert (np.abs(lse[seen] - l[seen]) <= (d + 2.0 ** -20 * (1 + np.abs(np.where(seen, l, 0))))[seen]).all()


def shared(rng, heads, dim, bs, lens, pool, wide=0, holes=0, pow2=True):
    """A cache of few blocks, which sequences of any length share (attention and selection only read); also ties."""
    k = rng.integers(-127, 128, (pool, heads, bs, dim), dtype=np.int8)
    v = rng.integers(-127, 128, (pool, heads, dim, bs), dtype=np.int8)
    scale = 2.0 ** rng.integers(-9, -4, (pool, heads, 2)) if pow2 else rng.uniform(0.005, 0.03, (pool, heads, 2))
    table = np.full((len(lens), max(wide, max(-(-n // bs) for n in lens), 1)), -1, np.int32)
    for row, n in zip(table, lens):
        used = -(-n // bs)
        row[:used] = rng.integers(0, pool, used)
        row[:used][rng.random(used) < holes] = rng.choice([-1, -7, pool, 2 ** 31 - 1])
    t = [dev(k), dev(v), dev(scale.astype(np.float32)), dev(np.stack((k.max(2), k.min(2)), 2))]
    return kv.KVCache(*t), table


def queries(rng, tokens, heads, dim, dt, aligned=True):
    """Rows that 16-byte loads can read, or slices of wider rows at odd addresses."""
    x = torch.from_numpy(rng.normal(size=(tokens, heads, dim))).to(dt).cuda()
    if aligned:
        return x
    wide = torch.zeros((tokens, heads, dim + 3), dtype=dt, device="cuda")
    wide[..., 1:dim + 1] = x
    return wide[..., 1:dim + 1]


# kv heads, group, dim, longest length, rows of each sequence: whether k_chunk takes them
RULE = [
    (8, 4, 128, 600, [48], False),               # work for a part of the chip
    (8, 4, 128, 8192, [64], True),
    (8, 4, 128, 8192, [10] * 32, False),         # too few rows
    (8, 4, 128, 8192, [1] * 64, False),          # single tokens, however they are passed
    (8, 4, 128, 8192, [512] + [1] * 63, False),
    (8, 4, 128, 8192, [2048] + [1] * 63, True),
    (8, 4, 256, 2048, [24] * 8, True),
    (8, 4, 256, 600, [24] * 8, False),
    (8, 4, 128, 128, [128] * 8, True),           # short prompts: many, and one
    (8, 4, 128, 256, [256], False),
    (8, 4, 64, 8192, [8], False),
    (8, 4, 192, 8192, [48] * 8, False),
    (8, 4, 192, 8192, [64] * 8, True),
    (8, 4, 64, 8192, [32] * 32, True),
]


@pytest.mark.parametrize("shape", RULE, ids=["%dx%d-%d-%d-%d" % (*s[:4], i) for i, s in enumerate(RULE)])
def test_which_kernel_takes_many_rows(shape):
    """The number of rows and the work decide, with or without the host's hint."""
    heads, group, dim, longest, news, chunk = shape
    rng = np.random.default_rng(35)
    lens = [longest] * len(news)
    cache, table = shared(rng, heads, dim, 64, lens, 60)
    off = offsets_of(news)
    q = torch.randn((off[-1], heads * group, dim), device="cuda").bfloat16()
    for hint in (None, max(news)):
        (got, lse), ran = launched(lambda: kv.attention(cache, q, dev(table), dev(np.int32(lens)), dev(off), max_tokens=hint,
                                                        return_lse=True))
        assert any("k_chunk" in x for x in ran) == chunk, ran
        check(Large(cache), got, lse, q, table, lens, off, dim ** -0.5)

# kv heads, group, dim, block tokens, type, lengths, rows of each, waves of a workgroup, table's width (0: as needed)
CHUNKS = [
    (1, 4, 128, 64, BF16, [200, 333, 0, 64], [200, 70, 3, 64], 4, 700),      # rows before the first token
    (2, 3, 96, 32, F16, [257, 31, 1], [257, 31, 1], 4, 700),
    (1, 2, 192, 16, BF16, [250, 195], [230, 195], 4, 2500),
    (1, 1, 256, 128, F16, [129, 400], [129, 90], 4, 400),
    (2, 5, 256, 64, BF16, [300, 77], [100, 77], 4, 200),
    (3, 1, 64, 16, BF16, [300, 20, 290], [300, 33, 90], 4, 1200),
    (1, 24, 128, 32, F16, [70, 9], [20, 12], 4, 1000),
    (1, 2, 64, 64, BF16, [5000, 4100], [140, 60], 4, 700),                   # over many tokens
    (9, 2, 64, 32, F16, [264, 130, 70], [264, 40, 70], 4, 400),
    (16, 1, 64, 16, BF16, [140 + 7 * i for i in range(9)], [140] * 9, 4, 900),
    (8, 2, 96, 32, BF16, [90 + 3 * i for i in range(16)], [90] * 16, 4, 400),
    (16, 1, 128, 128, F16, [600, 131, 130, 0, 1000, 128, 77, 500], [130, 131, 130, 1, 129, 128, 77, 500], 4, 0),
    (16, 1, 192, 64, BF16, [300] * 4 + [513, 270, 270, 261], [260] * 8, 4, 20),
    (16, 1, 256, 32, BF16, [300] * 4 + [513, 150, 150, 150], [150] * 8, 4, 0),
    (4, 2, 128, 16, BF16, [(37 * i) % 301 for i in range(70)], [(37 * i) % 301 for i in range(70)], 4, 0),  # 70 sequences
    (32, 1, 64, 64, F16, [520 + 9 * i for i in range(8)], [520] * 8, 8, 0),
    (32, 1, 96, 32, BF16, [520, 1, 700, 522, 523, 900, 519, 530], [520, 1, 700, 522, 523, 900, 519, 530], 8, 0),
    (8, 4, 128, 64, BF16, [520 + 64 * i for i in range(8)], [520] * 8, 8, 0),
]


@pytest.mark.parametrize("shape", CHUNKS, ids=["%dx%d-%d-%d-%s-%d" % (*s[:4], str(s[4])[6:], i) for i, s in enumerate(CHUNKS)])
@pytest.mark.parametrize("holes,scale,aligned", [(0, None, True), (0.1, 0.3, False), (0, -0.1, True)])
def test_prompts(shape, holes, scale, aligned):
    heads, group, dim, bs, dt, lens, news, waves, wide = shape
    rng = np.random.default_rng(30)
    cache, table = shared(rng, heads, dim, bs, lens, 40, wide, holes, scale is None)
    off = offsets_of(news)
    q = queries(rng, off[-1], heads * group, dim, dt, aligned)
    scale = scale or dim ** -0.5
    (got, lse), ran = launched(lambda: kv.attention(cache, q, dev(table), dev(np.int32(lens)), dev(off), scale=scale,
                                                    max_tokens=max(news), return_lse=True))
    kind = f"{dim}, {flag(dt == BF16)}"
    assert f"k_chunk<{kind}, {flag(aligned)}, {waves}>" in ran
    # few workgroups are split by the table's width
    assert bool(ran & {f"k_join<{kind}>", f"k_join_few<{kind}>"}) == (wide > 0 and heads * len(lens) < 128)
    check(Large(cache), got, lse, q, table, lens, off, scale)


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_many_splits(dim, dt):
    """Single tokens over long contexts, and lists of as many blocks: more splits than lanes read by themselves."""
    rng = np.random.default_rng(31)
    lens = [24001, 3, 0, 17000]
    cache, table = shared(rng, 1, dim, 64, lens, 300, holes=0.02)
    q = queries(rng, 4, 3, dim, dt) * 2
    off, n = offsets_of([1] * 4), dev(np.int32(lens))
    kind = f"{dim}, {flag(dt == BF16)}"
    (got, lse), ran = launched(lambda: kv.attention(cache, q, dev(table), n, return_lse=True))
    assert ran == {f"k_step<{kind}, false, true, 4>", f"k_join<{kind}>"}
    model = Large(cache)
    check(model, got, lse, q, table, lens, off, dim ** -0.5)
    lists = np.stack([rng.permutation(table.shape[1])[:330] for _ in lens]).astype(np.int32)[:, None]
    (got, lse), ran = launched(lambda: kv.sparse_attention(cache, q, dev(lists), dev(table), n, return_lse=True))
    assert ran == {f"k_step<{kind}, true, true, 4>", f"k_join<{kind}>"}
    check(model, got, lse, q, table, lens, off, dim ** -0.5, lists)


# kv heads, group, dim, type, lengths in blocks of 16, rows of each: the kernels
SELECTS = [
    (8, 4, 128, BF16, [1100 + 90 * i for i in range(10)], None, "k_select"),
    (8, 1, 64, F16, [300, 1, 0, 700, 1500, 2047, 64, 256, 257], None, "k_select"),
    (9, 5, 192, BF16, [520 + 40 * i for i in range(8)], None, "k_select"),
    (8, 2, 256, F16, [1030] * 9, None, "k_select"),
    (33, 17, 96, BF16, [1100, 900], None, "k_select"),
    (2, 16, 96, F16, [1300, 270], [20, 5], "k_select"),      # a chunk whose keys fill the LDS
    (2, 4, 128, BF16, [1300, 900], [20, 64], "k_select"),
    (1, 2, 192, BF16, [1300, 500], [40, 33], "k_select"),
    (2, 33, 64, F16, [700, 300], [3, 2], "k_select"),
    (1, 1, 256, BF16, [2000], [70], "k_select"),
    (1, 3, 128, F16, [1000, 2100, 800], None, "k_score"),    # few long rows
    (2, 2, 64, BF16, [24800, 30000], [3, 2], "k_score"),     # more keys than the LDS holds
    (1, 20, 192, F16, [25000], [2], "k_score"),
    (1, 1, 96, BF16, [24700], [66], "k_score"),
]


@pytest.mark.parametrize("shape", SELECTS, ids=["%dx%d-%d-%s-%d" % (*s[:3], str(s[3])[6:], i) for i, s in enumerate(SELECTS)])
@pytest.mark.parametrize("pow2,aligned", [(True, True), (False, False)])
def test_select(shape, pow2, aligned):
    heads, group, dim, dt, blocks, news, kernel = shape
    rng = np.random.default_rng(32)
    lens = [max(0, 16 * n - int(rng.integers(16))) for n in blocks]
    cache, table = shared(rng, heads, dim, 16, lens, 500, holes=0.02, pow2=pow2)
    off = offsets_of(news or [1] * len(lens))
    q = queries(rng, off[-1], heads * group, dim, dt, aligned)
    model = Large(cache)
    top = max(blocks)
    for count, sink, recent in ((1, 0, 0), (48, 1, 2), (700, 0, 3), (top + 5, 2, 0)):
        got, ran = launched(lambda: kv.select(cache, q, dev(table), dev(np.int32(lens)), count, dev(off) if news else None,
                                              sink=sink, recent=recent, max_tokens=max(news) if news else None))
        name = f"{kernel}<{dim}, {flag(dt == BF16)}, {flag(aligned)}>"
        assert ran == ({name, "k_top"} if kernel == "k_score" else {name})
        assert (got.cpu().numpy() == model.select(numbers(q), table, lens, off, count, sink, recent)).all()


@pytest.mark.parametrize("seqs", [64, 65, 130])
def test_many_sequences_of_few_rows(seqs):
    """Grids that go by the rows, over more sequences than a wave has lanes, some without rows."""
    rng = np.random.default_rng(33)
    heads, dim, bs = 2, 64, 16
    news = [int(x) for x in rng.choice([0, 0, 1, 1, 2, 40], seqs)]
    news[seqs // 2], news[-1] = 300, 3
    lens = [m + int(rng.integers(0, 50)) for m in news]
    wide = -(-max(lens) // bs)
    table, at = np.full((seqs, wide), -1, np.int32), 0
    ids = rng.permutation(sum(-(-n // bs) for n in lens) + 2)
    for row, n in zip(table, lens):
        used = -(-n // bs)
        row[:used] = ids[at:at + used]
        at += used
    cache = kv.KVCache.empty(len(ids), heads, dim, bs)
    cache.k.copy_(torch.from_numpy(rng.integers(-127, 128, cache.k.shape, dtype=np.int8)))
    cache.v.copy_(torch.from_numpy(rng.integers(-127, 128, cache.v.shape, dtype=np.int8)))
    cache.scale.fill_(2.0 ** -7)
    model = Large(cache)
    off = offsets_of(news)
    args = dev(table), dev(np.int32(lens)), dev(off)
    k, v = (torch.from_numpy(rng.normal(size=(off[-1], heads, dim))).to(BF16).cuda() for _ in range(2))
    kv.append(cache, k, v, *args, max_tokens=300)
    model.append(numbers(k), numbers(v), table, lens, off)
    for ids, n in zip(table, lens):  # behind a sequence's last token a block holds anything
        for j, at in enumerate(ids[:-(-n // bs)]):
            assert (numbers(cache.k[at])[:, :n - j * bs] == model.k[at][:, :n - j * bs]).all()
            assert (numbers(cache.v[at])[..., :n - j * bs] == model.v[at][..., :n - j * bs]).all()
    assert (numbers(cache.scale) == model.scale).all() and (cache.bound.cpu().numpy() == model.bound).all()
    q = queries(rng, off[-1], 3 * heads, dim, BF16)
    got, lse = kv.attention(cache, q, *args, max_tokens=300, return_lse=True)
    check(model, got, lse, q, table, lens, off, dim ** -0.5)
    chosen = kv.select(cache, q, args[0], args[1], 4, args[2], sink=1, recent=1, max_tokens=300)
    assert (chosen.cpu().numpy() == model.select(numbers(q), table, lens, off, 4, 1, 1)).all()
    got, lse = kv.sparse_attention(cache, q, chosen, *args, max_tokens=300, return_lse=True)
    check(model, got, lse, q, table, lens, off, dim ** -0.5, chosen.cpu().numpy())


# dim, type, with lists, waves of a workgroup
STEPS = [(d, dt, lists, waves) for d, dt in ((64, F16), (96, BF16), (128, F16), (192, BF16), (256, F16))
         for lists in (False, True) for waves in (4, 8)]


@pytest.mark.parametrize("shape", STEPS, ids=["%d-%s-%s-%d" % (s[0], str(s[1])[6:], s[2], s[3]) for s in STEPS])
def test_few_rows_at_odd_addresses(shape):
    dim, dt, listed, waves = shape
    rng = np.random.default_rng(34)
    lens, news = ([300, 33, 9, 2], [2, 1, 1, 3]) if waves == 8 else ([5000, 333, 9, 70], [3, 15, 9, 3])
    cache, table = shared(rng, 5, dim, 32, lens, 50, holes=0.05)
    off = offsets_of(news)
    q = queries(rng, off[-1], 5 * 7, dim, dt, False)
    args = dev(table), dev(np.int32(lens)), dev(off)
    lists = None
    if listed:
        lists = np.stack([rng.permutation(table.shape[1])[:9 if waves == 8 else 150] for _ in range(off[-1] * 5)])
        lists = lists.astype(np.int32).reshape(off[-1], 5, -1)
        (got, lse), ran = launched(lambda: kv.sparse_attention(cache, q, dev(lists), *args, return_lse=True))
    else:
        (got, lse), ran = launched(lambda: kv.attention(cache, q, *args, max_tokens=max(news), return_lse=True))
    assert f"k_step<{dim}, {flag(dt == BF16)}, {flag(listed)}, false, {waves}>" in ran
    check(Large(cache), got, lse, q, table, lens, off, dim ** -0.5, lists)
