"""Compaction of blocks whose products come near the end of float32's range or pass it, against the definition
(include/dance_kv_pages.h): x is code times scale in float32, what is not finite counts for no scale and takes the code
+-127, or 0 where it is no number. Everything has to be equal."""
import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, Model, codes_of, dev, make, scale_of

pytestmark = pytest.mark.gpu


def product(codes, scale):
    with np.errstate(over="ignore", invalid="ignore"):
        return np.float32(codes) * np.float32(scale)


def block_of(x):
    """Scale and codes of values [tokens, dim]."""
    a = np.abs(x.astype(np.float64))
    s = scale_of(float(a[np.isfinite(a)].max(initial=0.0)))
    with np.errstate(invalid="ignore"):
        return s, codes_of(x.astype(np.float64), s)


def check_compact(cache, table, tokens, keep):
    """keep: positions [kv heads, n]; into blocks of no sequence."""
    heads, bs, dim = cache.kv_heads, cache.block_tokens, cache.dim
    n = keep.shape[1]
    free = np.setdiff1d(np.arange(cache.blocks), table)[:-(-n // bs)].astype(np.int32)
    was = Model(cache)
    kv.compact(cache, dev(keep[None].astype(np.int32)), dev(np.int32([n])), dev(table), dev(np.int32([tokens])), dev(free[None]))
    now = Model(cache)
    for h in range(heads):
        at, slot = table[0, keep[h] // bs], keep[h] % bs
        k = product(was.k[at, h, slot], was.scale[at, h, 0, None])
        v = product(was.v[at, h, :, slot], was.scale[at, h, 1, None])
        for j, p in enumerate(free):
            part = slice(j * bs, min(n, (j + 1) * bs))
            for i, (x, got) in enumerate(((k[part], now.k[p, h]), (v[part], now.v[p, h].T))):
                s, codes = block_of(x)
                assert now.scale[p, h, i] == s
                assert np.array_equal(got[:len(codes)], codes) and not got[len(codes):].any()
                if i == 0:
                    assert np.array_equal(now.bound[p, h], np.stack((codes.max(0), codes.min(0))))


# powers of two of which a code's product passes the range, others, both signs of a mixture
SCALES = [[2.0 ** 122, 1.0], [1e37, 1.0], [2.0 ** 121, 2.0 ** 122], [2.7e36, 2.0 ** 120], [3.3e38, 2.0 ** 127],
          [2.0 ** 122, np.inf], [np.nan, 2.0 ** 123]]


@pytest.mark.parametrize("dim,bs", [(64, 16), (96, 128), (128, 64), (192, 32), (256, 16)])
@pytest.mark.parametrize("scales", SCALES)
@pytest.mark.parametrize("mixed", [False, True])
def test_products_beyond_the_range(dim, bs, scales, mixed):
    """Blocks of one scale, and tokens of two blocks in turn; each head in an order of its own."""
    rng = np.random.default_rng(60)
    cache, table = make(rng, 2, dim, bs, [2 * bs], spare=4)
    cache.scale[torch.from_numpy(table[0, :2]).long()] = torch.tensor(scales, device="cuda").float()[:, None, None]
    keep = np.stack([rng.permutation(2 * bs) if mixed else np.arange(2 * bs)[::1 - 2 * h] for h in range(2)])
    check_compact(cache, table, 2 * bs, keep)


def test_the_largest_finite_product_is_one_small_code():
    """A token whose other codes all pass the range, beside tokens of small scales: that code alone sets the block's scale."""
    rng = np.random.default_rng(61)
    cache, table = make(rng, 1, 64, 16, [16], spare=3)
    p = int(table[0, 0])
    cache.k[p], cache.v[p] = 127, -127
    cache.k[p, :, 5, 9], cache.v[p, :, 9, 5] = -3, 3
    cache.scale[p] = 2.0 ** 122
    check_compact(cache, table, 16, np.arange(16)[None])


def test_compact_after_append_of_the_largest_numbers():
    """append takes the scale 2^122 for bfloat16's largest number, whose code 64 stands for an infinity in float32, and
    2^121 or 2^122 for those next to it."""
    rng = np.random.default_rng(62)
    cache, table = make(rng, 2, 64, 16, [64], spare=6)
    top = float(torch.finfo(BF16).max)
    x = rng.uniform(-1, 1, (2, 64, 2, 64)) * top
    x[:, 3, :, 7], x[:, 20, :, 1] = top, -top * 0.99
    x[:, 16:48] *= 0.9
    x[:, 48:] = 0
    x[:, 50, :, 6], x[:, 50, :, 7] = top / 2, -top  # beside the largest one number that counts
    k, v = (torch.from_numpy(y).to(BF16).cuda() for y in x)
    kv.append(cache, k, v, dev(table), dev(np.int32([64])), dev(np.int32([0, 64])))
    assert float(cache.scale[torch.from_numpy(table[0, :4]).long()].max()) == 2.0 ** 122
    check_compact(cache, table, 64, np.stack([np.arange(64)[::2], np.arange(64)[::-2] ^ 1]))
    check_compact(cache, table, 64, np.stack([np.arange(48, 64)] * 2))
