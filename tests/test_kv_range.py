"""The key-value cache operators at the ends of their ranges: values and scales, numbers of
tokens, and the kernels that only large calls reach. Definitions and tolerances: test_kv.py."""
import math

import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, F16, Model, check_attention, dev, fake, make, numbers, offsets_of

# tokens over which a block repeats, sequences, rows of each, block tokens and dim: what joins the sums
LONG = [
    (40000, 1, 1, 128, 64),     # k_step, many splits: k_join
    (70000, 128, 1, 128, 64),   # k_step, few splits: k_join_few
    (140000, 1100, 1, 64, 64),  # k_step, one split
    (40000, 1, 200, 128, 128),  # k_step, many splits of many row tiles
    (140000, 256, 100, 64, 64),  # k_chunk, one split
    (40000, 1, 300, 128, 256),  # k_chunk, one wave a SIMD
    (40000, 1, 500, 128, 128),  # k_chunk, many splits
    (140000, 256, 130, 64, 64),  # k_chunk, one split, two row tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LONG, ids=["-".join(map(str, s)) for s in LONG])
@pytest.mark.parametrize("values", ["empty", "zeros", "tiny"])
def test_sums_over_long_contexts_of_least_values(shape, values):
    """Heads whose values are zero or of the least scale: the weights' sum is that of the keys alone.
    All tokens lie in one block, which the table repeats."""
    n, seqs, rows, bs, dim = shape
    rng = np.random.default_rng(20)
    cache = kv.KVCache.empty(1, 1, dim, bs)
    cache.k.copy_(torch.from_numpy(rng.integers(-127, 128, (1, 1, bs, dim), dtype=np.int8)))
    cache.scale[..., 0] = 2.0 ** -10
    if values != "empty":
        cache.scale[..., 1] = 2.0 ** -100
    if values == "tiny":
        cache.v.copy_(torch.from_numpy(rng.integers(-127, 128, (1, 1, dim, bs), dtype=np.int8)))
    table = torch.zeros((seqs, -(-n // bs)), dtype=torch.int32, device="cuda")
    q = torch.from_numpy(rng.normal(size=(seqs * rows, 1, dim))).to(BF16).cuda()
    q[0] = 0.0
    got, lse = kv.attention(cache, q, table, dev(np.full(seqs, n, np.int32)), dev(offsets_of([rows] * seqs)), scale=0.1,
                            max_tokens=rows, return_lse=True)
    # p whole blocks and r tokens of the last one
    seen = n - rows + 1 + np.arange(seqs * rows) % rows
    p, r = seen // bs, seen % bs
    keys, vals = numbers(cache.k)[0, 0] * 2.0 ** -10, numbers(cache.v)[0, 0].T * 2.0 ** -100
    x = numbers(q)[:, 0] @ keys.T * 0.1
    weight = np.exp(x) * (p[:, None] + (np.arange(bs) < r[:, None]))
    total = weight.sum(1)
    d = (np.abs(numbers(q)[:, 0]) @ np.abs(keys).T).max(1) * 0.1 * (dim + 8) * 2.0 ** -24
    want = np.log(total)
    assert (np.abs(numbers(lse)[:, 0] - want) <= d + 2.0 ** -20 * (1 + np.abs(want))).all()
    o, absolute = weight @ vals / total[:, None], weight @ np.abs(vals) / total[:, None]
    tol = 2.0 ** -8 * np.abs(o) + (2.0 ** -11 + 2 * d[:, None] + 2.0 ** -18) * absolute
    assert (np.abs(numbers(got)[:, 0] - o) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("e", [-100, -60, 100, 119, 120])
def test_values_of_the_least_and_the_largest_scales(e, rows):
    rng = np.random.default_rng(21)
    lens = [700, 70]
    cache, table = make(rng, 2, 128, 32, lens)
    cache.scale[..., 1] = 2.0 ** e
    off = offsets_of([rows] * 2)
    q = torch.from_numpy(rng.normal(size=(off[-1], 4, 128))).to(BF16).cuda()
    got, lse = kv.attention(cache, q, dev(table), dev(np.int32(lens)), dev(off), max_tokens=rows, return_lse=True)
    check_attention(Model(cache), got, lse, q, table, lens, off, 128 ** -0.5)

@pytest.mark.gpu
def test_prompt_of_more_rows_than_a_join_takes():
    """131,072 tokens of 64 heads, 2^23 rows: nothing is joined, so that only the kernel's own grid counts."""
    rng = np.random.default_rng(23)
    n, heads, dim, bs = 131072, 64, 64, 16
    cache, table = make(rng, 1, dim, bs, [bs])
    at = table[0, 0]
    g = torch.Generator(device="cuda").manual_seed(23)
    q = torch.randn((n, heads, dim), generator=g, device="cuda").to(BF16)
    got, lse = kv.attention(cache, q, dev(table[:, :1]), dev(np.int32([n])), dev(np.int32([0, n])), return_lse=True)
    keys = cache.k[at, 0].double() * cache.scale[at, 0, 0]
    vals = (cache.v[at, 0].double() * cache.scale[at, 0, 1]).t().contiguous()
    step = 8192
    for t in range(0, n, step):
        x = q[t:t + step].double().view(-1, dim)
        logits = x @ keys.t().contiguous() * dim ** -0.5
        pos = torch.arange(t, t + step, device="cuda").repeat_interleave(heads)
        logits.masked_fill_(torch.arange(bs, device="cuda") > pos[:, None], -math.inf)
        want = torch.logsumexp(logits, 1)
        p = torch.exp(logits - want[:, None])
        d = (x.abs() @ keys.abs().t().contiguous()).amax(1) * dim ** -0.5 * (dim + 8) * 2.0 ** -24
        o, absolute = p @ vals, p @ vals.abs()
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2 * d[:, None] + 2.0 ** -18) * absolute
        assert ((got[t:t + step].double().view(-1, dim) - o).abs() <= tol).all()
        assert ((lse[t:t + step].double().view(-1) - want).abs() <= d + 2.0 ** -20 * (1 + want.abs())).all()


def test_batches_too_large_for_a_launch_are_refused(capfd):
    c, b, r = fake(seqs=1, tokens=1 << 30, max_tokens=1 << 30, table_width=1)
    assert kv._bind().dance_kv_attention(c, b, r, 1.0, 1 << 20, None, 1 << 20, 1 << 60, None) == -1
    assert "too large for one launch" in capfd.readouterr().err

@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_logits_of_small_codes(dim, dt):
    """Blocks whose scale an outlier set: their other codes are small, and a logit is no less exact for it."""
    rng = np.random.default_rng(22)
    lens = [1, 2, 17, 64, 700]
    cache, table = make(rng, 2, dim, 32, lens)
    cache.k.copy_(torch.from_numpy(np.rint(rng.normal(size=cache.k.shape)).astype(np.int8)))
    cache.scale[..., 0] = 0.5
    q = torch.from_numpy(rng.normal(size=(5, 6, dim)) + 2).to(dt).cuda()
    got, lse = kv.attention(cache, q, dev(table), dev(np.int32(lens)), return_lse=True)
    check_attention(Model(cache), got, lse, q, table, lens, offsets_of([1] * 5), dim ** -0.5)
    lists = np.tile(np.arange(22, dtype=np.int32), (5, 2, 1))
    got, lse = kv.sparse_attention(cache, q, dev(lists), dev(table), dev(np.int32(lens)), return_lse=True)
    check_attention(Model(cache), got, lse, q, table, lens, offsets_of([1] * 5), dim ** -0.5, lists)
