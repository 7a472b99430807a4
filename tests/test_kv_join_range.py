"""Joins of rows at the end of their type's range. The weights exp(l_i - l) sum to 1, so that a joined row of finite parts is
finite, whatever its parts' sum would be. Tolerance: test_kv_parts.py."""
import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, F16, dev
from test_kv_parts import check_join

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("dim", [128, 7])
@pytest.mark.parametrize("count", [1, 2, 3, 5, 8])
def test_join_of_the_largest_numbers(dt, dim, count):
    """Parts of the type's largest numbers, of one sign and of both, with equal and other weights."""
    rng = np.random.default_rng(70 + count)
    top, tokens, heads = float(torch.finfo(dt).max), 12, 2
    parts, lses = [], []
    for _ in range(count):
        x = np.full((tokens, heads, dim), top)
        x[4:8] *= rng.choice([-1, 1], (4, heads, dim))
        x[8:] *= rng.uniform(-1, 1, (4, heads, dim))
        s = rng.normal(size=(tokens, heads))
        s[::2] = 3.5
        parts.append(torch.from_numpy(x).to(dt).cuda())
        lses.append(dev(np.float32(s)))
    got, lse = kv.join(parts, lses, return_lse=True)
    assert torch.isfinite(got).all() and (got[:4] == top).all()
    check_join(parts, lses, [None] * count, got, lse)
