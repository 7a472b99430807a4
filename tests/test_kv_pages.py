"""Owners, copies and compaction of the cache's blocks (include/dance_kv_pages.h, dance_amd/kv.py) against their
definitions in plain Python and numpy. All results are whole numbers, codes or powers of two and
have to be equal."""
import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, F16, Model, codes_of, dev, fake, make, numbers, offsets_of, scale_of


# ------------------------------------------------------------- definitions

class Owners:
    """A table, its lengths and the counts of its blocks' owners, and what the calls make of them."""

    def __init__(self, blocks, bs, table, lengths, pinned=()):
        self.blocks, self.bs = blocks, bs
        self.table, self.lengths = [list(map(int, row)) for row in table], list(map(int, lengths))
        self.refs = [0] * blocks
        for p in [p for row in self.table for p in row] + list(pinned):
            if 0 <= p < blocks:
                self.refs[p] += 1

    def width(self):
        return len(self.table[0])

    def owned(self, p):
        return 0 <= p < self.blocks

    def change(self, p, by):
        if self.owned(p):
            self.refs[p] += by

    def fork(self, parents):
        old, lens, n = self.table, self.lengths, len(self.table)
        for row in old:
            for p in row:
                self.change(p, -1)
        self.table = [list(old[p]) if 0 <= p < n else [-1] * len(old[0]) for p in parents]
        self.lengths = [lens[p] if 0 <= p < n else 0 for p in parents]
        for row in self.table:
            for p in row:
                self.change(p, 1)

    def reserve(self, upto):
        bs, refs = self.bs, list(self.refs)
        grows = [n < u <= self.width() * bs for n, u in zip(self.lengths, upto)]
        ends = [self.table[b][n // bs] if grows[b] and n % bs else -1 for b, n in enumerate(self.lengths)]
        free = [p for p in range(self.blocks) if refs[p] == 0]
        asked, now, src, dst = 0, [], [], []
        for b, (n, u) in enumerate(zip(list(self.lengths), upto)):
            pair, places, keeper = (-1, -1), [], False
            if grows[b]:
                for j in range(n // bs, (u - 1) // bs + 1):
                    p = self.table[b][j]
                    shared = self.owned(p) and refs[p] > 1
                    if j == n // bs and n % bs:
                        same = [c for c, e in enumerate(ends) if e == p]
                        keeper = shared and same[-1] == b and len(same) == refs[p]
                        if shared and not keeper:
                            places.append(j)
                    elif shared or not self.owned(p):
                        places.append(j)
            asked += len(places)
            served = grows[b] and (asked <= len(free) or not (places or keeper))
            if served:
                for j, q in zip(places, free[asked - len(places):]):
                    if j == n // bs and n % bs:
                        pair = (self.table[b][j], q)
                    self.change(self.table[b][j], -1)
                    self.change(q, 1)
                    self.table[b][j] = q
                self.lengths[b] = u
            now.append(u if served else n if u <= n else 0)
            src.append(pair[0])
            dst.append(pair[1])
        return now, src, dst

    def release(self, keep, start):
        for b, row in enumerate(self.table):
            lo, hi = 0, len(row)
            if keep is not None:
                self.lengths[b] = min(self.lengths[b], max(0, keep[b]))
                hi = -(-self.lengths[b] // self.bs)
            if start is not None:
                lo = max(0, start[b]) // self.bs
            for j in range(len(row)):
                if j < lo or j >= hi:
                    self.change(row[j], -1)
                    row[j] = -1


class Both:
    """The definitions and the library's calls, step by step."""

    def __init__(self, model):
        self.m = model
        self.pages = kv.Pages(dev(np.int32(model.refs)), model.bs)
        self.table, self.lengths = dev(np.int32(model.table)), dev(np.int32(model.lengths))

    def same(self):
        assert self.table.tolist() == self.m.table
        assert self.lengths.tolist() == self.m.lengths
        assert self.pages.refs.tolist() == self.m.refs

    def fork(self, parents):
        self.m.fork(parents)
        self.table, self.lengths = kv.fork(self.pages, self.table, self.lengths, dev(np.int32(parents)))
        self.same()

    def reserve(self, upto):
        want = self.m.reserve(upto)
        got = kv.reserve(self.pages, self.table, self.lengths, dev(np.int32(upto)))
        assert [x.tolist() for x in got] == [list(x) for x in want]
        self.same()
        return got

    def release(self, keep=None, start=None):
        self.m.release(keep, start)
        ints = [None if x is None else dev(np.int32(x)) for x in (keep, start)]
        kv.release(self.pages, self.table, self.lengths, *ints)
        self.same()


def owners(rng, seqs, width, bs, blocks, most, holes=0, pinned=0):
    """Sequences of random lengths in random blocks, as far as the pool reaches."""
    ids = rng.permutation(blocks).tolist()
    table, lens = np.full((seqs, width), -1, np.int64), []
    for b in range(seqs):
        n = int(rng.integers(0, most + 1))
        if -(-n // bs) > len(ids):
            n = 0
        for j in range(-(-n // bs)):
            table[b, j] = ids.pop()
        lens.append(n)
    for _ in range(holes):
        table[rng.integers(seqs), rng.integers(width)] = rng.choice([-1, -5, blocks, 2 ** 31 - 1])
    return Owners(blocks, bs, table, lens, [ids.pop() for _ in range(min(pinned, len(ids)))])


# --------------------------------------------------- owners: fork, reserve, release

# sequences, width, block tokens, blocks, longest, holes, pinned
POOLS = [(1, 1, 16, 1, 16, 0, 0), (1, 3, 128, 5, 300, 0, 1), (5, 7, 16, 40, 100, 0, 2), (8, 9, 32, 64, 200, 6, 0),
         (33, 5, 64, 130, 300, 0, 3), (70, 70, 16, 1500, 900, 20, 4), (3, 1500, 16, 5000, 20000, 5, 0),
         (300, 4, 16, 1025, 60, 0, 0), (9, 130, 16, 300000, 2000, 0, 9),
         # at the ends of what one workgroup takes, and beyond each
         (64, 1024, 16, 16384, 2000, 9, 5), (65, 1024, 16, 16384, 2000, 9, 5), (64, 1025, 16, 16384, 2000, 9, 5),
         (64, 1024, 16, 16385, 2000, 9, 5), (64, 3, 16, 70, 40, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("pool", POOLS, ids=["-".join(map(str, p)) for p in POOLS])
def test_owners_through_many_steps(pool):
    seqs, width, bs, blocks, most, holes, pinned = pool
    rng = np.random.default_rng(seqs * 1000 + width)
    both = Both(owners(rng, seqs, width, bs, blocks, most, holes, pinned))
    for step in range(12):
        parents = rng.integers(0, len(both.m.table), len(both.m.table))
        if step % 3 == 0:  # nobody moves, or slots end
            parents = np.where(rng.random(len(parents)) < 0.8, np.arange(len(parents)), rng.choice([-1, 2 ** 30]))
        both.fork(parents.tolist())
        grow = rng.integers(0, 2 + int(rng.choice([1, 3, bs, 3 * bs])), len(both.m.table))
        both.reserve([n + int(g) for n, g in zip(both.m.lengths, grow)])
        if step % 2:
            keep = [n - int(x) for n, x in zip(both.m.lengths, rng.integers(0, bs, len(both.m.table)))]
            both.release(keep=keep, start=None if step % 4 == 1 else [n - int(rng.integers(0, 3 * bs)) for n in keep])
        elif step % 4 == 2:
            both.release(start=[int(rng.integers(-5, most)) for _ in both.m.lengths])
    both.release(keep=[0] * len(both.m.table))
    assert both.m.refs.count(0) >= both.m.blocks - pinned


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 2, 7, 700])
def test_fork_to_other_numbers_of_rows(new):
    rng = np.random.default_rng(new)
    both = Both(owners(rng, 6, 2100, 16, 9000, 20000))
    both.fork(rng.integers(-1, 7, new).tolist())
    both.fork([0] * 5)
    both.fork([4])


@pytest.mark.gpu
def test_last_owner_keeps_a_partly_filled_block():
    both = Both(Owners(8, 16, [[3, -1]], [10]))
    both.fork([0, 0, 0])
    now, src, dst = both.reserve([11, 11, 11])
    assert src.tolist() == [3, 3, -1] and dst.tolist() == [0, 1, -1] and both.pages.refs.tolist() == [1, 1, 0, 1, 0, 0, 0, 0]
    both.fork([0, 0, 1])
    now, src, dst = both.reserve([11, 12, 12])  # one of two owners grows: it copies
    assert src.tolist() == [-1, 0, -1] and now.tolist() == [11, 12, 12]


@pytest.mark.gpu
def test_pool_without_room():
    # three free blocks; the second sequence needs two, the third two
    both = Both(Owners(6, 16, [[0, -1, -1], [1, -1, -1], [2, -1, -1], [-1, -1, -1]], [16, 16, 16, 0]))
    now, _, _ = both.reserve([17, 48, 17, 0])
    assert now.tolist() == [17, 48, 0, 0] and both.lengths.tolist() == [17, 48, 16, 0]
    now, _, _ = both.reserve([18, 40, 17, 1])  # without free blocks: what needs none goes on
    assert now.tolist() == [18, 48, 0, 0]
    now, _, _ = both.reserve([49, 49, 1 << 30, 0])  # beyond the table
    assert now.tolist() == [0, 0, 0, 0]
    # all owners of a block grow and only one has room for a copy: the last one may not write what another still reads
    both = Both(Owners(2, 16, [[0, -1]], [5]))
    both.fork([0, 0, 0])
    now, src, dst = both.reserve([6, 6, 6])
    assert now.tolist() == [6, 0, 0] and src.tolist() == [0, -1, -1] and dst.tolist() == [1, -1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [30, 20000])  # one launch and two
def test_reserve_of_nothing_and_of_what_is_there(blocks):
    """Lengths that stay, go back or are no lengths; the same tensor for both; sequences that end on a block's last place."""
    both = Both(Owners(blocks, 16, [[3, 4, -1], [5, -1, -1], [-1, -1, -1], [6, 7, 8], [-1, -1, -1]], [32, 16, 0, 41, 0]))
    now, src, dst = both.reserve([32, 10, 0, -7, -2 ** 31])
    assert now.tolist() == [32, 16, 0, 41, 0] and src.tolist() == [-1] * 5
    kv.reserve(both.pages, both.table, both.lengths, both.lengths)
    both.same()
    now, _, _ = both.reserve([33, 17, 48, 48, 49])
    assert now.tolist() == [33, 17, 48, 48, 0]
    both.release(keep=both.m.lengths)
    kv.release(both.pages, both.table, both.lengths, keep=both.lengths)
    both.same()
    both.release(start=[2 ** 31 - 1, 16, -2 ** 31, 31, 0])


@pytest.mark.gpu
def test_blocks_that_the_caller_keeps():
    """One more owner for the blocks of a prompt: they outlive every sequence, and the partly filled one is always copied."""
    both = Both(Owners(12, 16, [[2, 5, -1]], [20]))
    for p in (2, 5):
        both.m.refs[p] += 1
        both.pages.refs[p] += 1
    both.fork([0, 0, -1])
    now, src, dst = both.reserve([21, 21, 0])
    assert src.tolist() == [5, 5, -1] and dst.tolist() == [0, 1, -1] and now.tolist() == [21, 21, 0]
    both.release(keep=[0, 0, 0])
    assert both.m.refs == [0, 0, 1, 0, 0, 1] + [0] * 6


@pytest.mark.gpu
def test_places_reserved_ahead():
    """Room for more than is written: later calls find it, forks of it get their own."""
    both = Both(Owners(64, 16, [[9, -1, -1, -1, -1]], [3]))
    both.reserve([70])
    both.release(keep=[20])
    both.reserve([33])
    both.fork([0, 0])
    both.release(keep=[40, 40])
    both.reserve([41, 60])
    both.release(keep=[0, 60])


# ---------------------------------------------------------------- copy

def pools(rng, layers, heads, dim, bs, blocks):
    out = []
    for _ in range(layers):
        c = kv.KVCache.empty(blocks, heads, dim, bs)
        for t in (c.k, c.v, c.bound):
            t.copy_(dev(rng.integers(-128, 128, t.shape, dtype=np.int8)))
        c.scale.copy_(dev(rng.random(c.scale.shape)))
        out.append(c)
    return out


def arrays(c):
    return [c.k, c.v, c.scale, c.bound]


@pytest.mark.gpu
@pytest.mark.parametrize("layers,heads,dim,bs,pairs", [(1, 1, 64, 16, 1), (3, 5, 96, 32, 9), (40, 2, 128, 16, 6), (2, 3, 192, 128, 20),
                                                       (1, 1, 64, 16, 2500), (2, 7, 256, 64, 5)])
@pytest.mark.parametrize("other", [False, True])
def test_copy(layers, heads, dim, bs, pairs, other):
    rng = np.random.default_rng(pairs)
    blocks = 2 * pairs + 3
    caches = pools(rng, layers, heads, dim, bs, blocks)
    into = pools(rng, layers, heads, dim, bs, pairs + 2) if other else caches
    src = rng.integers(0, pairs + 3, pairs)
    dst = rng.permutation(pairs) if other else pairs + 3 + rng.permutation(pairs)
    for x in (src, dst):  # pairs that are none
        x[rng.random(pairs) < 0.3] = rng.choice([-1, blocks, 2 ** 31 - 1, -2 ** 31])
    want = [[a.clone() for a in arrays(c)] for c in into]
    for c, w in zip(caches, want):
        for a, x in zip(arrays(c), w):
            for s, d in zip(src, dst):
                if 0 <= s < blocks and 0 <= d < len(x):
                    x[d] = a[s]
    kv.copy(caches if layers > 1 else caches[0], dev(np.int32(src)), dev(np.int32(dst)), into=into if other else None)
    for c, w in zip(into, want):
        assert all(torch.equal(a, x) for a, x in zip(arrays(c), w))


@pytest.mark.gpu
def test_copy_of_layers_in_one_array():
    """Layers whose scales begin at any multiple of 8 bytes."""
    rng, shape = np.random.default_rng(11), (4, 5, 3)  # layers, blocks, heads
    k, v, b = (dev(rng.integers(-128, 128, shape + x, dtype=np.int8)) for x in ((16, 64), (64, 16), (2, 64)))
    s = dev(np.float32(rng.random(shape + (2,))))
    want = [x.clone() for x in (k, v, s, b)]
    for x in want:
        x[:, 4] = x[:, 1]
    kv.copy([kv.KVCache(k[i], v[i], s[i], b[i]) for i in range(4)], dev(np.int32([1, -1])), dev(np.int32([4, 0])))
    assert all(torch.equal(x, y) for x, y in zip((k, v, s, b), want))


@pytest.mark.gpu
def test_copy_and_compact_beyond_32_bit_offsets():
    heads, bs, dim = 8, 128, 256
    blocks = (1 << 32) // (heads * bs * dim) + 40
    cache = kv.KVCache.empty(blocks, heads, dim, bs)
    rng = np.random.default_rng(3)
    small = pools(rng, 1, heads, dim, bs, 4)[0]
    small.scale.copy_(dev(2.0 ** rng.integers(-9, -4, small.scale.shape)))
    far = [blocks - 1, blocks - 2, blocks - 20, 5]
    kv.copy(small, dev(np.int32([0, 1, 2, 3])), dev(np.int32(far)), into=cache)
    keep = dev(np.int32(rng.permutation(500)[:300].reshape(1, 1, -1)))
    n, m = dev(np.int32([500])), dev(np.int32([300]))
    other = kv.KVCache.empty(3, heads, dim, bs)
    kv.compact(small, keep, m, dev(np.int32([[0, 1, 2, 3]])), n, dev(np.int32([[0, 1, 2]])), into=other)
    kv.compact(cache, keep, m, dev(np.int32([far])), n, dev(np.int32([[blocks - 5, 1, blocks - 9]])))
    for a, b in zip(arrays(cache), arrays(other)):
        assert torch.equal(a[[blocks - 5, 1, blocks - 9]], b)


# -------------------------------------------------------------- compact

def compacted(model, keep, counts, table, lengths, into_table, into):
    """The definition, on a Model of the cache written into (its arrays change)."""
    heads, bs, dim = model.heads, model.bs, model.dim
    out = []
    for b, n in enumerate(counts):
        for j in range(min(into_table.shape[1], -(-min(n, keep.shape[2]) // bs))):
            p, live = into_table[b, j], min(bs, min(n, keep.shape[2]) - j * bs)
            if not 0 <= p < into.blocks:
                continue
            for h in range(heads):
                x = np.zeros((2, bs, dim), np.float32)
                for i in range(live):
                    at = keep[b, h % keep.shape[1], j * bs + i]
                    if not 0 <= at < min(lengths[b], table.shape[1] * bs) or not model.has(table[b, at // bs]):
                        continue
                    q = table[b, at // bs]
                    s = model.scale[q, h].astype(np.float32)
                    x[0, i] = model.k[q, h, at % bs].astype(np.float32) * s[0]
                    x[1, i] = model.v[q, h, :, at % bs].astype(np.float32) * s[1]
                s = [scale_of(float(np.abs(y).max())) for y in x]
                k, v = (codes_of(y.astype(np.float64), t) for y, t in zip(x, s))
                out.append((p, h, k, v.T, s, (k[:live].max(0), k[:live].min(0))))
    for p, h, k, v, s, bound in out:
        into.k[p, h], into.v[p, h], into.scale[p, h], into.bound[p, h] = k, v, s, bound


# kv heads, dim, block tokens, lengths, counts, heads with lists of their own
COMPACT = [
    (2, 128, 64, [700, 64, 65, 0], [333, 64, 1, 0], True),
    (1, 64, 16, [1, 17, 40], [1, 16, 17], True),
    (3, 96, 32, [200, 33], [90, 33], False),
    (2, 192, 128, [300, 129], [129, 127], True),
    (5, 256, 64, [321], [200], True),
    (1, 96, 128, [128, 500], [128, 255], True),
    (4, 64, 128, [1000], [130], False),
    (2, 256, 16, [90, 31], [31, 16], True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", COMPACT, ids=[f"{s[0]}-{s[1]}-{s[2]}-{i}" for i, s in enumerate(COMPACT)])
@pytest.mark.parametrize("pow2,other", [(True, True), (False, False)])
def test_compact(shape, pow2, other):
    heads, dim, bs, lens, counts, own = shape
    rng = np.random.default_rng(dim + bs)
    need = sum(-(-n // bs) for n in counts)
    cache, table = make(rng, heads, dim, bs, lens, holes=2, spare=need + 4, pow2=pow2)
    into = make(rng, heads, dim, bs, [bs * need])[0] if other else cache
    free = rng.permutation(into.blocks) if other else np.setdiff1d(np.arange(cache.blocks), table)
    wide = max(-(-n // bs) for n in counts) + 1
    into_table, at = np.full((len(lens), wide), -1, np.int32), 0
    for b, n in enumerate(counts):
        w = -(-n // bs)
        into_table[b, :w] = free[at:at + w]
        at += w
    if len(counts) > 1:
        into_table[0, 0] = into.blocks + 7  # a hole among the new places
    keep = np.full((len(lens), heads if own else 1, max(counts) + 3), -1, np.int32)
    for b, (n, m) in enumerate(zip(lens, counts)):
        for h in range(keep.shape[1]):
            keep[b, h, :m] = np.sort(rng.permutation(max(n, 1))[:m]) if h % 2 == 0 else rng.integers(0, max(n, 1), m)
    keep[0, 0, :3] = [-1, lens[0], 2 ** 31 - 1]  # tokens that are not there
    model, target = Model(cache), Model(into)
    kv.compact(cache, dev(keep), dev(np.int32(counts)), dev(table), dev(np.int32(lens)), dev(into_table),
               into=into if other else None)
    compacted(model, keep, counts, table, lens, into_table, target)
    got, written = Model(into), np.setdiff1d(into_table, [-1, into.blocks + 7])
    for name in ("k", "v", "scale", "bound"):
        a, b = getattr(got, name), getattr(target, name)
        assert np.array_equal(a[written], b[written]), name
        assert np.array_equal(a, b, equal_nan=name == "scale"), name


@pytest.mark.gpu
def test_compact_counts_beyond_the_lists_and_the_table():
    rng = np.random.default_rng(5)
    cache, table = make(rng, 2, 64, 16, [100], spare=6)
    free = np.setdiff1d(np.arange(cache.blocks), table)
    keep = np.sort(rng.permutation(100)[:40]).astype(np.int32).reshape(1, 1, 40)
    for count, wide in ((1 << 30, 3), (40, 2), (-3, 3)):
        model, target = Model(cache), Model(cache)
        into = np.int32([free[:wide]])
        kv.compact(cache, dev(keep), dev(np.int32([count])), dev(table), dev(np.int32([100])), dev(into))
        compacted(model, keep, [max(count, 0)], table, [100], into, target)
        got = Model(cache)
        assert np.array_equal(got.k, target.k) and np.array_equal(got.v, target.v) and np.array_equal(got.bound, target.bound)


@pytest.mark.gpu
@pytest.mark.parametrize("scales", [[2.0 ** -100, 2.0 ** 100], [1e-38, 2.0 ** 60], [np.nan, 1.0], [np.inf, 1.0]])
def test_compact_of_far_apart_scales(scales):
    """A block of the least scale beside one of a large; scales that are no numbers."""
    rng = np.random.default_rng(6)
    cache, table = make(rng, 1, 64, 16, [32], spare=4)
    cache.scale[torch.from_numpy(table[0, :2]).long()] = torch.tensor(scales, device="cuda").float()[:, None, None]
    free = np.int32([np.setdiff1d(np.arange(cache.blocks), table)[:2]])
    keep = np.arange(0, 32, dtype=np.int32).reshape(1, 1, 32)[..., ::-1].copy()
    x = {i: cache.k[int(table[0, i]), 0].double().cpu().numpy() * float(np.float32(s)) for i, s in enumerate(scales)}
    kv.compact(cache, dev(keep), dev(np.int32([32])), dev(table), dev(np.int32([32])), dev(free))
    for j, i in ((0, 1), (1, 0)):
        y = x[i][::-1]
        with np.errstate(invalid="ignore"):
            y = np.float32(y)
        finite = np.abs(y[np.isfinite(y)])
        step = scale_of(float(finite.max(initial=0.0)))
        assert float(cache.scale[int(free[0, j]), 0, 0]) == step
        assert np.array_equal(numbers(cache.k[int(free[0, j]), 0]), codes_of(y.astype(np.float64), step))


@pytest.mark.gpu
def test_compact_of_the_least_code():
    """-128, which append never writes, needs the next scale: 127 steps would not hold it."""
    rng = np.random.default_rng(7)
    cache, table = make(rng, 1, 64, 16, [16], spare=3)
    p, free = int(table[0, 0]), int(np.setdiff1d(np.arange(cache.blocks), table)[0])
    cache.k[p], cache.v[p], cache.scale[p] = -128, -128, 0.25
    cache.k[p, :, 3], cache.v[p, :, :, 5] = 127, 1
    keep = dev(np.arange(16, dtype=np.int32).reshape(1, 1, 16))
    kv.compact(cache, keep, dev(np.int32([16])), dev(table), dev(np.int32([16])), dev(np.int32([[free]])))
    assert (cache.scale[free] == 0.5).all()
    k, v = cache.k[free, 0], cache.v[free, 0]
    assert (k[3] == 64).all() and (k[4] == -64).all() and (v[:, 5] == 0).all() and (v[:, 4] == -64).all()  # halves to even
    assert (cache.bound[free, 0, 0] == 64).all() and (cache.bound[free, 0, 1] == -64).all()


# ------------------------------------------------------- as they are used together

@pytest.mark.gpu
@pytest.mark.parametrize("dt,bs,dim", [(BF16, 16, 64), (F16, 32, 96)])
def test_beams_that_share_blocks_equal_beams_that_do_not(dt, bs, dim):
    """A beam search over two layers: prompts fork, beams are chosen anew at every step and grow by a token or
    by a draft of which some is given back. Beside it every beam keeps all of its blocks to itself, copied
    whole at every choice: codes and attention have to be equal."""
    rng, beams, heads, steps = np.random.default_rng(bs), 6, 2, 14
    width, blocks = 9, 60
    shared = [kv.KVCache.empty(blocks, heads, dim, bs) for _ in range(2)]
    alone = [kv.KVCache.empty(2 * beams * width, heads, dim, bs) for _ in range(2)]
    pages = kv.Pages.empty(blocks, bs)
    prompts = np.int32([3 * bs + 5, 2 * bs])
    table, lengths = dev(np.full((2, width), -1, np.int32)), dev(np.int32([0, 0]))
    own = np.arange(beams * width, dtype=np.int32).reshape(beams, width)
    spare = own + beams * width

    def rows(n):
        return [torch.from_numpy(rng.normal(size=(n, heads, dim)) * np.exp(rng.normal(size=(n, 1, 1)))).to(dt).cuda() for _ in range(4)]

    now, src, dst = kv.reserve(pages, table, lengths, dev(prompts))
    assert now.tolist() == prompts.tolist()
    off = offsets_of(prompts)
    x = rows(off[-1])
    for i in range(2):
        kv.append(shared[i], x[2 * i], x[2 * i + 1], table, now, dev(off))
        kv.append(alone[i], x[2 * i], x[2 * i + 1], dev(own[[0, 1]]), now, dev(off))
    parents = [0, 0, 0, 1, 1, 1]
    lens = prompts.copy()
    for step in range(steps):
        table, lengths = kv.fork(pages, table, lengths, dev(np.int32(parents)))
        for i in range(2):
            kv.copy(alone[i], dev(own[parents].reshape(-1)), dev(spare.reshape(-1)))
        own, spare = spare, own
        lens = lens[parents]
        grow = [1, 1, 2, 1][step % 4]
        now, src, dst = kv.reserve(pages, table, lengths, lengths + grow)
        kv.copy(shared, src, dst)
        assert now.tolist() == (lens + grow).tolist()
        off = offsets_of([grow] * beams)
        x = rows(off[-1])
        q = torch.from_numpy(rng.normal(size=(off[-1], 2 * heads, dim))).to(dt).cuda()
        for i in range(2):
            kv.append(shared[i], x[2 * i], x[2 * i + 1], table, now, dev(off))
            kv.append(alone[i], x[2 * i], x[2 * i + 1], dev(own), now, dev(off))
            a, b = (kv.attention(c, q, t, now, dev(off)) for c, t in ((shared[i], table), (alone[i], dev(own))))
            assert torch.equal(a, b), step
        lens = lens + grow
        if grow == 2:
            lens = lens - 1
            kv.release(pages, table, lengths, keep=dev(np.int32(lens)))
        assert lengths.tolist() == lens.tolist()
        refs = np.bincount(table.cpu().numpy()[table.cpu().numpy() >= 0], minlength=blocks)
        assert refs.tolist() == pages.refs.tolist()
        parents = rng.integers(0, beams, beams).tolist()
    kv.release(pages, table, lengths, keep=dev(np.zeros(beams, np.int32)))
    assert not pages.refs.any() and not lengths.any() and (table == -1).all()


@pytest.mark.gpu
def test_eviction_keeps_what_is_attended_to():
    """Half of the tokens move to new blocks, the old ones are given back; attention sees the kept tokens."""
    rng, heads, dim, bs = np.random.default_rng(8), 2, 128, 32
    lens, counts = np.int32([300, 65]), np.int32([150, 33])
    cache = kv.KVCache.empty(40, heads, dim, bs)
    pages = kv.Pages.empty(40, bs)
    table, lengths = dev(np.full((2, 12), -1, np.int32)), dev(np.int32([0, 0]))
    now, _, _ = kv.reserve(pages, table, lengths, dev(lens))
    k, v = (torch.from_numpy(rng.normal(size=(365, heads, dim))).to(F16).cuda() for _ in range(2))
    kv.append(cache, k, v, table, now, dev(offsets_of(lens)))
    keep = np.zeros((2, heads, 150), np.int32)
    for b in range(2):
        for h in range(heads):
            keep[b, h, :counts[b]] = np.sort(rng.permutation(lens[b])[:counts[b]])
    before, old = Model(cache), table.cpu().numpy()
    fresh, none = dev(np.full((2, 12), -1, np.int32)), dev(np.int32([0, 0]))
    now, _, _ = kv.reserve(pages, fresh, none, dev(counts))
    assert now.tolist() == counts.tolist()
    kv.compact(cache, dev(keep), now, table, lengths, fresh)
    kv.release(pages, table, lengths, keep=dev(np.int32([0, 0])))
    assert int(pages.refs.sum()) == 5 + 2
    after, t = Model(cache), fresh.cpu().numpy()
    for b in range(2):
        for h in range(heads):
            for i in range(counts[b]):
                at, p = keep[b, h, i], t[b, i // bs]
                src = old[b, at // bs]
                for new, was, c in ((after.k[p, h, i % bs], before.k[src, h, at % bs], 0),
                                    (after.v[p, h, :, i % bs], before.v[src, h, :, at % bs], 1)):
                    d = np.abs(new * after.scale[p, h, c] - was * before.scale[src, h, c])
                    assert (d <= after.scale[p, h, c] / 2).all()  # within half a step of the new scale


@pytest.mark.gpu
def test_graph_of_a_serving_step_replays():
    """fork, reserve, copy, append, attention and release in one graph, over tensors that stay: the table and the
    lengths go back into them at the end."""
    rng, seqs, heads, dim, bs, blocks, width = np.random.default_rng(9), 4, 2, 64, 16, 64, 8

    def state():
        return dict(caches=[kv.KVCache.empty(blocks, heads, dim, bs) for _ in range(2)], pages=kv.Pages.empty(blocks, bs),
                    table=dev(np.full((seqs, width), -1, np.int32)), lengths=dev(np.zeros(seqs, np.int32)),
                    parents=dev(np.arange(seqs, dtype=np.int32)), back=dev(np.zeros(seqs, np.int32)),
                    x=torch.zeros((2 * seqs, 8, dim), dtype=BF16, device="cuda"))

    off = dev(np.arange(0, 2 * seqs + 1, 2, dtype=np.int32))

    def step(s):
        table, lengths = kv.fork(s["pages"], s["table"], s["lengths"], s["parents"])
        now, src, dst = kv.reserve(s["pages"], table, lengths, lengths + 2)
        kv.copy(s["caches"], src, dst)
        out = []
        for c in s["caches"]:
            kv.append(c, s["x"][:, 4:6], s["x"][:, 6:], table, now, off)
            out.append(kv.attention(c, s["x"][:, :4], table, now, off))
        kv.release(s["pages"], table, lengths, keep=lengths - s["back"])
        s["table"].copy_(table)
        s["lengths"].copy_(lengths)
        return now, src, dst, *out

    captured, eager = state(), state()
    step(state())  # the library is loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(captured)
    for s in (captured,):  # capturing runs nothing, but the state starts from the same place all the same
        assert not s["lengths"].any()
    for i in range(20):
        parents = rng.integers(0, seqs, seqs) if i else np.zeros(seqs)
        if i == 9:
            parents = np.full(seqs, -1)
        back, x = rng.integers(0, 3, seqs), rng.normal(size=(2 * seqs, 8, dim))
        for s in (captured, eager):
            s["parents"].copy_(torch.from_numpy(np.int32(parents)))
            s["back"].copy_(torch.from_numpy(np.int32(back)))
            s["x"].copy_(torch.from_numpy(x))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        assert torch.equal(captured["table"], eager["table"]) and torch.equal(captured["pages"].refs, eager["pages"].refs)


@pytest.mark.gpu
def test_page_calls_run_on_the_current_stream():
    rng = np.random.default_rng(10)
    model = owners(rng, 5, 9, 16, 40, 100)
    want, both = Both(model), None
    start = [x.clone() for x in (want.pages.refs, want.table, want.lengths)]
    upto = [n + 20 for n in model.lengths]
    want.fork([1, 1, 2, 3, 0])
    want.reserve(upto)
    want.release(keep=[n - 3 for n in upto])
    refs, table, lengths = (torch.zeros_like(x) for x in start)
    parents, up, keep = (dev(np.int32(x)) for x in ([1, 1, 2, 3, 0], upto, [n - 3 for n in upto]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-4
        for a, b in zip((refs, table, lengths), start):
            a.copy_(b)
        pages = kv.Pages(refs, 16)
        table, lengths = kv.fork(pages, table, lengths, parents)
        kv.reserve(pages, table, lengths, up)
        kv.release(pages, table, lengths, keep=keep)
    torch.cuda.current_stream().wait_stream(side)
    assert refs.tolist() == want.m.refs and table.tolist() == want.m.table and lengths.tolist() == want.m.lengths


# ------------------------------------------------------------- refusals

@pytest.mark.gpu
def test_refusals():
    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")
    cache, other = kv.KVCache.empty(4, 2, 64, 16), kv.KVCache.empty(4, 2, 64, 32)
    pages, t, n = kv.Pages.empty(4, 16), ints(3, 2), ints(3)
    for exc, call in [
            (TypeError, lambda: kv.Pages(ints(4).long())),
            (TypeError, lambda: kv.Pages(ints(4, 1))),
            (ValueError, lambda: kv.Pages(ints(0))),
            (ValueError, lambda: kv.Pages(ints(8)[::2])),
            (ValueError, lambda: kv.Pages(ints(4), 48)),
            (ValueError, lambda: kv.Pages(ints(4).cpu())),
            (ValueError, lambda: kv.fork(pages, t[0], n, n)),
            (ValueError, lambda: kv.fork(pages, t[:0], n[:0], n)),
            (ValueError, lambda: kv.fork(pages, t, n[:2], n)),
            (ValueError, lambda: kv.fork(pages, t, n, n[:0])),
            (TypeError, lambda: kv.fork(pages, t, n, n.long())),
            (ValueError, lambda: kv.fork(pages, t, n, n.cpu())),
            (TypeError, lambda: kv.reserve(pages, t.long(), n, n)),
            (ValueError, lambda: kv.reserve(pages, t.t(), n[:2], n[:2])),
            (ValueError, lambda: kv.reserve(pages, t, n, n[:1])),
            (ValueError, lambda: kv.release(pages, t, n, keep=n[:1])),
            (TypeError, lambda: kv.release(pages, t, n, start=n.float())),
            (ValueError, lambda: kv.copy([], n, n)),
            (ValueError, lambda: kv.copy(cache, n, n[:2])),
            (TypeError, lambda: kv.copy(cache, n.long(), n)),
            (ValueError, lambda: kv.copy([cache, other], n, n)),
            (ValueError, lambda: kv.copy(cache, n, n, into=other)),
            (ValueError, lambda: kv.copy([cache, cache], n, n, into=[cache])),
            (ValueError, lambda: kv.copy([cache, kv.KVCache.empty(5, 2, 64, 16)], n, n)),
            (ValueError, lambda: kv.compact(cache, ints(3, 2, 5), n, t, n, t, into=other)),
            (ValueError, lambda: kv.compact(cache, ints(3, 3, 5), n, t, n, t)),
            (ValueError, lambda: kv.compact(cache, ints(3, 2, 0), n, t, n, t)),
            (ValueError, lambda: kv.compact(cache, ints(3, 5), n, t, n, t)),
            (TypeError, lambda: kv.compact(cache, ints(3, 2, 5).long(), n, t, n, t)),
            (ValueError, lambda: kv.compact(cache, ints(2, 2, 5), n, t, n, t)),
            (ValueError, lambda: kv.compact(cache, ints(3, 2, 5), n[:2], t, n, t)),
            (ValueError, lambda: kv.compact(cache, ints(3, 2, 5), n, t, n, t[:2])),
            (ValueError, lambda: kv.compact(cache, ints(3, 2, 5), n, t, n, t[0]))]:
        with pytest.raises(exc):
            call()
    kv.copy(cache, n[:0], n[:0])
    kv.release(pages, t, n)
    assert not pages.refs.any()


@pytest.mark.parametrize("header,count", [("dance_kv_pages.h", 6), ("dance_kv_parts.h", 3)])
def test_headers_are_c_and_their_entries_are_exported(header, count):
    import re
    import subprocess
    import dance_amd as D
    path = D.HERE + "/../include/" + header
    for lang in ("c", "c++"):
        subprocess.run(["gcc", "-x", lang, "-fsyntax-only", "-Wall", "-Wextra", "-Werror", path], check=True)
    names = set(re.findall(r"\b(dance_kv_\w+)\(const", open(path).read()))
    assert len(names) == count
    out = subprocess.run(["nm", "-D", "--defined-only", D.LIB_PATH], capture_output=True, text=True).stdout
    assert {n for n in names if f" T {n}\n" in out} == names


def test_entries_refuse_before_any_device_work(capfd):
    """Pointers that are never followed: every call is refused on the host."""
    L, p = kv._bind(), 1 << 20

    def pages(refs=p, blocks=8, block_tokens=16):
        return kv.DanceKvPages(refs, blocks, block_tokens)

    calls = []
    for bad in (pages(None), pages(blocks=0), pages(blocks=1 << 31), pages(block_tokens=24), None):
        calls += [(L.dance_kv_fork, [bad, p, p, 2, 3, p, 2, p + 64, p + 64, None]),
                  (L.dance_kv_reserve, [bad, p, p, 2, 3, p, p, p, p, p, 1 << 30, None]),
                  (L.dance_kv_release, [bad, p, p, 2, 3, p, p, None])]
        assert L.dance_kv_reserve_work(bad, 2, 3) == 0
    ok, large = pages(), pages(blocks=1 << 20)
    assert L.dance_kv_reserve_work(ok, 2, 3) == 0  # one workgroup's
    need = L.dance_kv_reserve_work(large, 2, 3)
    assert need == (1 << 17) + 2 * 8 + 2 * 4 + 4096
    for seqs, width in ((0, 3), (2, 0), (2, 1 << 28)):
        calls += [(L.dance_kv_fork, [ok, p, p, seqs, width, p, 2, p + 64, p + 64, None]),
                  (L.dance_kv_reserve, [ok, p, p, seqs, width, p, p, p, p, p, 1 << 30, None]),
                  (L.dance_kv_release, [ok, p, p, seqs, width, p, p, None])]
    for i in (1, 2, 5, 7, 8):
        args = [ok, p, p, 2, 3, p, 2, p + 64, p + 64, None]
        args[i] = None
        calls.append((L.dance_kv_fork, args))
    calls += [(L.dance_kv_fork, [ok, p, p, 2, 3, p, 0, p + 64, p + 64, None]),
              (L.dance_kv_fork, [ok, p, p, 2, 3, p, 2, p, p + 64, None]),
              (L.dance_kv_fork, [ok, p, p, 2, 3, p, 2, p + 64, p, None]),
              (L.dance_kv_fork, [ok, p, p, 1 << 24, 1 << 10, p, 2, p + 64, p + 64, None])]  # more threads than a launch has
    for i in (1, 2, 5, 6, 7, 8, 9):
        args = [large, p, p, 2, 3, p, p, p, p, p, need, None]
        args[i] = None
        calls.append((L.dance_kv_reserve, args))
    calls += [(L.dance_kv_reserve, [large, p, p, 2, 3, p, p, p, p, p, need - 1, None]),
              (L.dance_kv_reserve, [large, p, p, 2, 3, p, p, p, p, p + 8, need, None]),
              (L.dance_kv_reserve, [ok, p, p, 1 << 20, 1 << 12, p, p, p, p, p, 1 << 50, None]),
              (L.dance_kv_release, [ok, None, p, 2, 3, p, p, None]), (L.dance_kv_release, [ok, p, None, 2, 3, p, p, None])]
    c = fake()[0]
    for change in ({"k": None}, {"scale": p | 4}, {"bound": p | 8}, {"dim": 100}, {"block_tokens": 8}, {"blocks": 0}, {"kv_heads": 0}):
        bad = fake(**change)[0]
        calls += [(L.dance_kv_copy, [bad, c, 1, p, p, 2, None]), (L.dance_kv_copy, [c, bad, 1, p, p, 2, None]),
                  (L.dance_kv_compact, [bad, c, p, p, 2, 3, p, 2, 5, p, p, 3, None]),
                  (L.dance_kv_compact, [c, bad, p, p, 2, 3, p, 2, 5, p, p, 3, None])]
    for change in ({"kv_heads": 4}, {"dim": 128}, {"block_tokens": 32}):
        bad = fake(**change)[0]
        calls += [(L.dance_kv_copy, [bad, c, 1, p, p, 2, None]), (L.dance_kv_compact, [c, bad, p, p, 2, 3, p, 2, 5, p, p, 3, None])]
    two = (kv.DanceKvCache * 2)(c, fake(blocks=5)[0])
    calls += [(L.dance_kv_copy, [None, c, 1, p, p, 2, None]), (L.dance_kv_copy, [c, None, 1, p, p, 2, None]),
              (L.dance_kv_copy, [c, c, 0, p, p, 2, None]), (L.dance_kv_copy, [c, c, 1, None, p, 2, None]),
              (L.dance_kv_copy, [c, c, 1, p, None, 2, None]), (L.dance_kv_copy, [two, two, 2, p, p, 2, None])]
    for i in (2, 3, 6, 9, 10):
        args = [c, c, p, p, 2, 3, p, 2, 5, p, p, 3, None]
        args[i] = None
        calls.append((L.dance_kv_compact, args))
    for i, x in ((4, 0), (5, 0), (7, 3), (8, 0), (11, 0), (5, 1 << 28), (4, 1 << 30)):
        args = [c, c, p, p, 2, 3, p, 2, 5, p, p, 3, None]
        args[i] = x
        calls.append((L.dance_kv_compact, args))
    wide = fake(dim=256, block_tokens=128)[0]  # 512 threads a block: 2^33 in all
    calls.append((L.dance_kv_compact, [wide, wide, p, p, 1 << 23, 3, p, 2, 128, p, p, 3, None]))
    for i, (fn, args) in enumerate(calls):
        capfd.readouterr()
        assert fn(*args) == -1, (i, fn.__name__, args)
        assert fn.__name__ in capfd.readouterr().err, (i, fn.__name__, args)
    assert L.dance_kv_copy(c, c, 1, None, None, 0, None) == 0  # no pairs: nothing to do
    assert L.dance_kv_release(ok, p, p, 2, 3, None, None, None) == 0


@pytest.mark.gpu
def test_example_of_beam_decoding():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv_beams.py")
    spec = importlib.util.spec_from_file_location("kv_beams", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.run(users=3, beams=4, prompt=1500, steps=20, layers=2, heads=8, kv_heads=2, block_tokens=32, quiet=True)
    assert len(got) == 20 and all(r["missed"] == 0 and r["owned"] <= r["named"] for r in got)
    # three roundings to bfloat16 and the weights' to 11 bits, of outputs of about one size: a few 2^-9 of their norm
    assert all(r["apart"] < 2.0 ** -6 for r in got)
    assert got[-1]["left"] == sum(-(-((1500 - 331 * u + 21) // 2) // 32) for u in range(3))
