"""Attention over parts of a context (include/dance_kv_parts.h, dance_amd/kv.py): rows that see all of another
sequence, and joined attentions, against their definitions in 64 bits on the CPU.

Cross attention has attention's tolerance (test_kv.py). A joined row is sum w_i o_i / sum w_i with w_i =
exp(l_i - m): each weight is off by at most e_i = 2^-21 + |l_i - m| 2^-23 of itself (the difference's rounding, the
exponential's within 4 units, products and sums of eight parts with 2^-24 each), once above and once below, so the row by
u |o| + 2 sum w_i e_i |o_i| / sum w_i + half the least number of its type, and its logarithm by 2^-23 |l| + 2 max
w_i e_i + 2^-22."""
import math

import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, F16, IDS, LEAST, PROMPTS, ROUND, SHAPES, Model, check_attention, dev, fake, make, numbers, offsets_of
from test_kv_paths import launched


def check_cross(model, got, lse, q, table, lens, off, scale):
    """Every row as a sequence of its own, whose last token it is."""
    seq = np.repeat(np.arange(len(lens)), np.diff(off))
    check_attention(model, got, lse, q, table[seq], [min(lens[b], table.shape[1] * model.bs) for b in seq],
                    np.arange(len(seq) + 1), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("holes", [0, 2])
def test_cross_attention(shape, holes):
    heads, group, dim, bs, dt, lens, news = shape
    rng = np.random.default_rng(31)
    cache, table = make(rng, heads, dim, bs, lens, holes)
    off = offsets_of(news or [1] * len(lens))
    q = torch.from_numpy(rng.normal(size=(off[-1], heads * group, dim))).to(dt).cuda()
    got, lse = kv.cross_attention(cache, q, dev(table), dev(np.int32(lens)), dev(off) if news else None, return_lse=True,
                                  max_tokens=max(news) if news else None)
    check_cross(Model(cache), got, lse, q, table, lens, off, dim ** -0.5)


# more rows than tokens, fewer, sequences without any, and lengths that the prompts' kernel takes
MANY = PROMPTS + [(2, 4, 128, 64, F16, [5, 0, 300], [90, 70, 40]), (1, 4, 64, 32, BF16, [1, 33], [130, 1]),
                  (1, 1, 192, 64, BF16, [700], [400]), (2, 8, 96, 16, F16, [2000, 17], [33, 64])]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MANY, ids=[f"{s[0]}x{s[1]}-{s[2]}-{s[3]}-{i}" for i, s in enumerate(MANY)])
@pytest.mark.parametrize("holes,scale", [(0, None), (3, 0.3), (0, -0.1), (0, 0.0)])
def test_cross_attention_of_many_rows(shape, holes, scale):
    heads, group, dim, bs, dt, lens, news = shape
    rng = np.random.default_rng(32)
    cache, table = make(rng, heads, dim, bs, lens, holes, pow2=scale is None)
    off = offsets_of(news)
    q = torch.from_numpy(rng.normal(size=(off[-1], heads * group, dim))).to(dt).cuda()
    got, lse = kv.cross_attention(cache, q, dev(table), dev(np.int32(lens)), dev(off), scale=scale, return_lse=True,
                                  max_tokens=max(news))
    check_cross(Model(cache), got, lse, q, table, lens, off, dim ** -0.5 if scale is None else scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_cross_attention_reads_no_other_tokens(dt):
    """What lies behind the last token, in other blocks and in holes changes nothing; rows have strides and odd addresses."""
    rng, heads, dim, bs = np.random.default_rng(33), 2, 64, 32
    lens, news = [40, 0, 95], [3, 2, 70]
    cache, table = make(rng, heads, dim, bs, lens)
    off = offsets_of(news)
    wide = torch.from_numpy(rng.normal(size=(off[-1], 3, 5, dim + 3))).to(dt).cuda()
    q = wide[:, 1, :4, 3:]
    args = dev(table), dev(np.int32(lens)), dev(off)
    want, lse = kv.cross_attention(cache, q.contiguous(), *args, return_lse=True)
    for b, n in enumerate(lens):
        if n % bs:
            p = int(table[b, n // bs])
            cache.k[p, :, n % bs:] = 127
            cache.v[p, :, :, n % bs:] = -127
    got, other = kv.cross_attention(cache, q, *args, return_lse=True)
    assert torch.equal(got, want) and torch.equal(lse, other)
    assert not want[3:5].any() and torch.isneginf(lse[3:5]).all() and torch.isfinite(lse[5:]).all()


# calls of each kind of plan: both kernels, in workgroups of four and eight waves, in splits joined both ways and in one
PLANS = [
    (2, 4, 128, 64, BF16, [5000], [64]),
    (8, 4, 128, 64, BF16, [3000, 2900, 10], [64, 200, 64]),
    (4, 1, 64, 32, F16, [9000], None),
    (16, 1, 64, 64, BF16, [1100] * 48, None),
    (16, 1, 96, 64, F16, [2100] * 6, [16] * 6),
    (4, 2, 192, 64, BF16, [2500, 7], [90, 33]),
    (2, 4, 256, 128, F16, [4000], [50]),
    (8, 8, 64, 16, BF16, [700, 650, 3], [130, 120, 128]),
    (1, 2, 256, 16, BF16, [6000], [3]),
    (4, 2, 64, 64, F16, [1990] * 35 + [5], None),
    (4, 4, 64, 64, BF16, [1990, 300] * 18, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", PLANS, ids=[f"{s[0]}x{s[1]}-{s[2]}-{len(s[5])}x{s[5][0]}" for s in PLANS])
def test_cross_attention_in_every_plan(shape):
    cache, table, q, off, call = plan_case(*shape)
    got, lse = call()
    check_cross_large(cache, got, lse, q, table, shape[5], off, shape[2] ** -0.5)


def plan_case(heads, group, dim, bs, dt, lens, news):
    rng = np.random.default_rng(35)
    cache, table = make(rng, heads, dim, bs, lens, holes=2)
    off = offsets_of(news or [1] * len(lens))
    q = torch.from_numpy(rng.normal(size=(off[-1], heads * group, dim))).to(dt).cuda()
    t, n, o = dev(table), dev(np.int32(lens)), dev(off) if news else None
    return cache, table, q, off, lambda: kv.cross_attention(cache, q, t, n, o, return_lse=True,
                                                            max_tokens=max(news) if news else None)


@pytest.mark.gpu
def test_plans_reach_every_kernel():
    """So that the shapes above are looked at again where the choice of plans changes."""
    ran = set()
    for shape in PLANS:
        ran |= launched(plan_case(*shape)[-1])[1]
    if not ran:
        pytest.skip("torch's profiler does not name the kernels here")
    kinds = {k.split("<")[0] + ("-" + k[:-1].split(", ")[-1] if "join" not in k else "") for k in ran}
    assert kinds == {"k_step-4", "k_step-8", "k_chunk-4", "k_chunk-8", "k_join", "k_join_cross", "k_join_few"}


def check_cross_large(cache, got, lse, q, table, lens, off, scale):
    """check_cross in products for each sequence and head, on the GPU in 64 bits; the tolerance is check_attention's."""
    group, dim = q.shape[1] // cache.kv_heads, cache.dim
    for b, n in enumerate(lens):
        rows, used = slice(off[b], off[b + 1]), -(-n // cache.block_tokens)
        ids = torch.from_numpy(table[b, :used].astype(np.int64)).cuda()
        live = (ids >= 0) & (ids < cache.blocks)
        seen = live.repeat_interleave(cache.block_tokens)[:n]
        ids = torch.where(live, ids, 0)
        for h in range(cache.kv_heads):
            s = cache.scale[ids, h].double()
            k = (cache.k[ids, h].double() * s[:, 0, None, None]).reshape(-1, dim)[:n][seen]
            v = (cache.v[ids, h].double() * s[:, 1, None, None]).transpose(1, 2).reshape(-1, dim)[:n][seen]
            for f in range(h * group, (h + 1) * group):
                if not len(k):
                    assert not got[rows, f].any() and torch.isneginf(lse[rows, f]).all()
                    continue
                x = q[rows, f].double()
                logits = x @ k.T * scale
                w = torch.softmax(logits, 1)
                o, absolute = w @ v, w @ v.abs()
                d = (x.abs() @ k.abs().T).amax(1) * abs(scale) * (dim + 8) * 2.0 ** -24
                tol = ROUND[q.dtype] * o.abs() + (2.0 ** -11 + 2 * d[:, None] + 2.0 ** -18) * absolute + LEAST[q.dtype] / 2
                assert ((got[rows, f].double() - o).abs() <= tol).all(), (b, f)
                l = torch.logsumexp(logits, 1)
                assert ((lse[rows, f].double() - l).abs() <= d + 2.0 ** -20 * (1 + l.abs())).all(), (b, f)


@pytest.mark.gpu
def test_cross_attention_near_attention_of_the_last_rows():
    """One row a sequence: both see all tokens, perhaps in other splits. Each is within attention's tolerance of the exact
    row, so they are within twice that of each other; its largest part here is the output's rounding and 2^-11 of the weights."""
    rng = np.random.default_rng(34)
    for dim, lens in ((128, [3000, 1, 64]), (256, [70000]), (64, [17] * 40)):
        cache, table = make(rng, 2, dim, 64, lens)
        q = torch.from_numpy(rng.normal(size=(len(lens), 8, dim))).to(BF16).cuda()
        args = cache, q, dev(table), dev(np.int32(lens))
        (a, l), (b, m) = kv.attention(*args, return_lse=True), kv.cross_attention(*args, return_lse=True)
        top = float((cache.v[torch.from_numpy(table[table >= 0]).long()].abs().amax((1, 2, 3))
                     * cache.scale[torch.from_numpy(table[table >= 0]).long()][..., 1].amax(1)).max())
        assert float((a.double() - b.double()).abs().max()) <= 2 * (2.0 ** -8 + 2.0 ** -10) * top
        assert float((l - m).abs().max()) <= 2.0 ** -10


# ---------------------------------------------------------------- join

def check_join(parts, lses, rows, got, lse):
    tokens, heads, dim = got.shape
    l, o = np.full((len(parts), tokens, heads), -np.inf), np.zeros((len(parts), tokens, heads, dim))
    for i, (p, s, r) in enumerate(zip(parts, lses, rows)):
        r = np.arange(tokens) if r is None else r.cpu().numpy()
        there = (r >= 0) & (r < len(p))
        l[i, there], o[i, there] = numbers(s)[r[there]], numbers(p)[r[there]]
    o = np.where(np.isneginf(l)[..., None], 0, o)
    m = l.max(0)
    some = np.isfinite(m)
    x = np.where(some, l - np.where(some, m, 0), -np.inf)
    w = np.exp(x)
    total = np.where(some, w.sum(0), 1)
    want = (w[..., None] * o).sum(0) / total[..., None]
    e = 2.0 ** -21 + np.where(np.isfinite(x), np.abs(x), 0) * 2.0 ** -23
    tol = (ROUND[got.dtype] * np.abs(want) + 2 * ((w * e)[..., None] * np.abs(o)).sum(0) / total[..., None]
           + LEAST[got.dtype] / 2)
    err = np.abs(numbers(got) - want)
    assert (err <= tol).all(), float((err - tol).max())
    if lse is not None:
        lse, want = numbers(lse), np.where(some, np.where(some, m, 0) + np.log(total), -np.inf)
        assert (np.isneginf(lse) == ~some).all()
        t = 2.0 ** -23 * np.abs(want) + 2 * (w * e).max(0) + 2.0 ** -22
        assert (np.abs(lse[some] - want[some]) <= t[some]).all()


def parts_of(rng, count, tokens, heads, dim, dt, some):
    parts, lses, rows = [], [], []
    for i in range(count):
        n, r = tokens, None
        if some and i % 2:
            n = max(1, tokens // 2)
            r = rng.integers(-2, n + 2, tokens)
            r[rng.random(tokens) < 0.1] = rng.choice([2 ** 31 - 1, -2 ** 31])
            r = dev(np.int32(r))
        parts.append(torch.from_numpy(rng.normal(size=(n, heads, dim)) * 10.0 ** rng.uniform(-3, 2)).to(dt).cuda())
        s = rng.normal(size=(n, heads)) * rng.choice([1, 8, 60]) + rng.choice([0, 300])
        s[rng.random(s.shape) < 0.2] = -np.inf
        lses.append(dev(np.float32(s)))
        rows.append(r)
    return parts, lses, rows


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("tokens,heads,dim,dt", [(1, 1, 64, BF16), (33, 6, 96, F16), (5, 3, 256, BF16), (70, 2, 7, F16), (3, 1, 2500, BF16),
                                                 (9, 1, 1, F16), (300, 32, 128, F16)])
@pytest.mark.parametrize("some", [False, True])
def test_join(count, tokens, heads, dim, dt, some):
    rng = np.random.default_rng(count * 100 + tokens)
    parts, lses, rows = parts_of(rng, count, tokens, heads, dim, dt, some)
    got, lse = kv.join(parts, lses, rows if some else None, return_lse=True)
    check_join(parts, lses, rows, got, lse)
    assert torch.equal(kv.join(parts, lses, rows), got)


@pytest.mark.gpu
def test_join_of_strided_parts_and_of_rows_that_count_for_nothing():
    rng, dt = np.random.default_rng(41), BF16
    wide = torch.from_numpy(rng.normal(size=(20, 2, 3, 67))).to(dt).cuda()
    parts = [wide[:, 0, :, 3:], wide[:, 1, :, :64], wide[:, :, 0, 1:65].transpose(0, 1)[1][:, None].expand(-1, 3, -1)]
    lses = [dev(np.float32(rng.normal(size=(20, 3)))) for _ in parts]
    got, lse = kv.join(parts, lses, return_lse=True)
    check_join(parts, lses, [None] * 3, got, lse)
    # NaN and infinities in rows that count for nothing
    bad = [p.clone() for p in parts]
    for i, x in enumerate((math.nan, math.inf)):
        lses[i][i::2] = -math.inf
        bad[i][i::2] = x
    clean = [torch.where(torch.isfinite(b), b, 0) for b in bad]
    got, lse = kv.join(bad, lses, return_lse=True)
    check_join(clean, lses, [None] * 3, got, lse)
    for s in lses:
        s[7] = -math.inf
    out = torch.full((20, 3, 64), 9.0, dtype=dt, device="cuda")
    assert kv.join(bad, lses, out=out) is out and not out[7].any() and torch.isfinite(out).all()


@pytest.mark.gpu
def test_join_of_logarithms_that_are_no_numbers():
    x = torch.ones((4, 1, 8), dtype=F16, device="cuda")
    a, b = (torch.tensor(v, device="cuda")[:, None] for v in ([math.nan, 1.0, math.nan, -math.inf], [1.0, math.nan, -math.inf, 2.0]))
    got, lse = kv.join([x, 2 * x], [a, b], return_lse=True)
    assert torch.isnan(got[:3]).all() and torch.isnan(lse[:3]).all() and (got[3] == 2).all() and float(lse[3]) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 90])
def test_cross_attention_in_a_wide_table(rows):
    """Blocks that a sequence has been given beyond its length count for nothing, with and without the longest length."""
    rng = np.random.default_rng(36)
    lens = [130, 64, 1]
    cache, table = make(rng, 2, 128, 32, lens, spare=60)
    wide = np.concatenate([table, np.setdiff1d(np.arange(cache.blocks), table)[:57].reshape(3, 19)], 1).astype(np.int32)
    wide = np.where((wide < 0) | (wide >= cache.blocks), wide[:, -1:], wide)
    off = offsets_of([rows] * 3)
    q = torch.from_numpy(rng.normal(size=(off[-1], 4, 128))).to(BF16).cuda()
    for longest in (None, 130):
        got, lse = kv.cross_attention(cache, q, dev(wide), dev(np.int32(lens)), dev(off), max_tokens=rows, max_length=longest,
                                      return_lse=True)
        check_cross(Model(cache), got, lse, q, table, lens, off, 128 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_shared_prefix_and_own_tokens_equal_the_whole(dt):
    """Sequences of two groups that share their group's prompt: the prompt's blocks are read once for a group's rows, each
    sequence's own behind them, and joined. Against attention over all of it in 64 bits: attention's roundings, those of the two parts (u of
    each, by weight) and the join's."""
    rng, heads, group, dim, bs = np.random.default_rng(42), 2, 4, 128, 32
    shared, each = [10, 3], [5, 4]  # blocks of the prompts, sequences of the groups
    lens = [s * bs + int(n) for s, c in zip(shared, each) for n in rng.integers(1, 100, c)]
    cache, full = make(rng, heads, dim, bs, lens)
    at = 0
    for s, c in zip(shared, each):
        full[at:at + c, :s] = full[at, :s]
        at += c
    skip = np.repeat(shared, each)
    own = np.full((len(lens), 5), -1, np.int32)
    for b, s in enumerate(skip):
        own[b, :min(5, full.shape[1] - s)] = full[b, s:s + 5]
    q = torch.from_numpy(rng.normal(size=(len(lens), heads * group, dim))).to(dt).cuda()
    prefix, l0 = kv.cross_attention(cache, q, dev(full[[0, each[0]], :10].copy()), dev(np.int32([s * bs for s in shared])),
                                    dev(offsets_of(each)), return_lse=True)
    rest, l1 = kv.attention(cache, q, dev(own), dev(np.int32(lens) - np.int32(skip * bs)), return_lse=True)
    got, lse = kv.join([prefix, rest], [l0, l1], return_lse=True)
    model = Model(cache)
    o, l, absolute, g = model.attention(numbers(q), full, lens, np.arange(len(lens) + 1), dim ** -0.5)
    d = g * (dim + 8) * 2.0 ** -24
    u = ROUND[dt]
    tol = u * np.abs(o) + (u * (1 + u) + 2.0 ** -11 + 2 * d[..., None] + 2.0 ** -18 + 2.0 ** -17) * absolute
    assert (np.abs(numbers(got) - o) <= tol).all()
    assert (np.abs(numbers(lse) - l) <= d + 2.0 ** -19 * (1 + np.abs(l))).all()


@pytest.mark.gpu
def test_graph_of_parts_replays():
    rng, heads, dim, bs = np.random.default_rng(43), 2, 64, 16
    cache, table = make(rng, heads, dim, bs, [500, 30, 90])
    prefix, t, n = dev(table[:1].copy()), dev(table), dev(np.int32([500, 30, 90]))
    long, off = dev(np.int32([500])), dev(np.int32([0, 3]))
    q = torch.zeros((3, 8, dim), dtype=F16, device="cuda")
    rows = dev(np.int32([0, -1, 2]))

    def step():
        a, l = kv.cross_attention(cache, q, prefix, long, off, return_lse=True)
        b, m = kv.attention(cache, q, t, n, return_lse=True)
        return kv.join([a, b], [l, m], [rows, None], return_lse=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(5):
        q.copy_(torch.from_numpy(rng.normal(size=q.shape)))
        n.copy_(dev(np.int32([rng.integers(1, 500), 30, rng.integers(0, 91)])))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_no_rows_and_other_streams():
    rng = np.random.default_rng(44)
    cache, table = make(rng, 1, 64, 16, [20])
    t, n = dev(table), dev(np.int32([20]))
    q = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    assert kv.cross_attention(cache, q, t, n, dev(np.int32([0, 0]))).shape == (0, 2, 64)
    got, lse = kv.join([q, q], [q.new_zeros((0, 2)).float()] * 2, return_lse=True)
    assert got.shape == (0, 2, 64) and lse.shape == (0, 2)
    empty = kv.join([q], [q.new_zeros((0, 2)).float()], [dev(np.int32([0, 5]))])  # a part without rows
    assert empty.shape == (2, 2, 64) and not empty.any()
    # behind work on another stream
    parts = [torch.from_numpy(rng.normal(size=(6, 2, 64))).to(BF16).cuda() for _ in range(2)]
    lses = [torch.zeros((6, 2), device="cuda") for _ in range(2)]
    want, late = kv.join(parts, lses), [torch.zeros_like(p) for p in parts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-4
        for a, b in zip(late, parts):
            a.copy_(b)
        got = kv.join(late, lses)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


# ------------------------------------------------------------- refusals

@pytest.mark.gpu
def test_refusals():
    cache = kv.KVCache.empty(4, 2, 64, 16)
    t, n = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros((3, 4, 64), dtype=BF16, device="cuda")
    lse = torch.zeros((3, 4), device="cuda")
    for exc, call in [
            (TypeError, lambda: kv.cross_attention(cache, q.float(), t, n)),
            (ValueError, lambda: kv.cross_attention(cache, q[:, :3], t, n)),
            (ValueError, lambda: kv.cross_attention(cache, q[:2], t, n)),
            (ValueError, lambda: kv.cross_attention(cache, q, t, n, n)),
            (ValueError, lambda: kv.cross_attention(cache, q, t, n, out=q[:2])),
            (RuntimeError, lambda: kv.cross_attention(cache, q, t, n, scale=math.inf)),
            (ValueError, lambda: kv.join([], [])),
            (ValueError, lambda: kv.join([q] * 9, [lse] * 9)),
            (ValueError, lambda: kv.join([q], [])),
            (ValueError, lambda: kv.join([q], [lse], [])),
            (ValueError, lambda: kv.join([q[0]], [lse[0]])),
            (ValueError, lambda: kv.join([q[:, :0]], [lse[:, :0]])),
            (TypeError, lambda: kv.join([q.float()], [lse])),
            (TypeError, lambda: kv.join([q, q.half()], [lse, lse])),
            (ValueError, lambda: kv.join([q, q[..., :32]], [lse, lse])),
            (ValueError, lambda: kv.join([q, q[:2]], [lse, lse[:2]])),
            (ValueError, lambda: kv.join([q.transpose(1, 2)], [lse])),
            (ValueError, lambda: kv.join([q.cpu()], [lse.cpu()])),
            (ValueError, lambda: kv.join([q, q.cpu()], [lse, lse])),
            (TypeError, lambda: kv.join([q], [lse.half()])),
            (ValueError, lambda: kv.join([q], [lse[:2]])),
            (ValueError, lambda: kv.join([q], [lse.t().contiguous().t()])),
            (TypeError, lambda: kv.join([q], [lse], [n.long()])),
            (ValueError, lambda: kv.join([q, q], [lse, lse], [None, n[:2]])),
            (ValueError, lambda: kv.join([q], [lse], [n[:0].view(0, 1)])),
            (ValueError, lambda: kv.join([q], [lse], out=q[:2]))]:
        with pytest.raises(exc):
            call()


def test_entries_refuse_before_any_device_work(capfd):
    """Pointers that are never followed: every call is refused on the host."""
    L, p = kv._bind(), 1 << 20
    for change in ({"k": None}, {"dim": 100}, {"table": None}, {"seqs": 0}, {"max_tokens": 6}, {"data": None}, {"heads": 3}, {"dtype": 0}):
        c, b, r = fake(**change)
        assert L.dance_kv_cross_attention(c, b, r, 1.0, p, None, p, 1 << 40, None) == -1
        assert "dance_kv_cross_attention" in capfd.readouterr().err
    c, b, r = fake(seqs=1, table_width=5000, tokens=1, max_tokens=1)
    r.heads = 2
    need = L.dance_kv_cross_attention_work(c, b, 2)
    assert need > 0 and L.dance_kv_cross_attention_work(c, b, 3) == 0 and L.dance_kv_cross_attention_work(c, b, 0) == 0
    for at, size in ((None, need), (p, need - 1), (p | 8, need)):
        assert L.dance_kv_cross_attention(c, b, r, 1.0, p, None, at, size, None) == -1
    assert L.dance_kv_cross_attention(c, b, r, math.nan, p, None, p, need, None) == -1
    assert L.dance_kv_cross_attention(c, b, r, 1.0, None, None, p, need, None) == -1

    def part(data=p, lse=p, rows=None, tokens=5):
        return kv.DanceKvPart(data, 256, 64, lse, rows, tokens)

    def join(parts, count=None, tokens=5, heads=4, dim=64, dtype=3, out=p):
        a = (kv.DanceKvPart * max(1, len(parts)))(*parts) if parts is not None else None
        return L.dance_kv_join(a, len(parts or []) if count is None else count, tokens, heads, dim, dtype, out, None, None)

    ok = part()
    for args in ([None], [[]], [[ok] * 9], [[part(None)]], [[part(p | 1)]], [[ok, part(lse=None)]], [[part(tokens=4)]],
                 [[part(rows=p, tokens=1 << 31)]]):
        assert join(*args) == -1
    for change in ({"heads": 0}, {"heads": 1 << 16}, {"dim": 0}, {"dim": 1 << 17}, {"dtype": 1}, {"out": None}, {"out": p | 1},
                   {"tokens": 4}):
        assert join([ok, ok], **change) == -1
    assert join([part(tokens=1 << 30)], tokens=1 << 30) == -1  # 2^32 rows
    assert join([part(None, None, None, 0)], tokens=0, out=None) == 0
    assert capfd.readouterr().err.count("dance_kv_join") == 8 + 8 + 1
