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
from test_kv import BF16, LEAST, ROUND, Model, dev, numbers, offsets_of

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
