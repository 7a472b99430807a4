"""Cross attention in calls that reach each kernel of the cache's attention at each of its dimensions, with both element
types, blocks smaller and larger than a tile, splits in one and joined in every way, and a sequence without tokens beside
long ones. A table's width decides the plan, so that rows times tokens can stay few. Every case names the kernels
that it means and asks torch's profiler which ran. Definitions and tolerance: test_kv_paths.py."""
import numpy as np
import pytest
import torch

from dance_amd import kv
from test_kv import BF16, F16, dev, offsets_of
from test_kv_paths import Large, check, flag, kernels_have_names, launched, queries, shared  # noqa: F401

pytestmark = pytest.mark.gpu


class Whole(Large):
    """Every row sees all of its sequence's tokens."""

    def attention(self, q, table, lengths, offsets, scale, lists=None):
        t, heads, dim = q.shape
        group = heads // self.heads
        out = [np.zeros((t, heads, dim)), np.full((t, heads), -np.inf), np.zeros((t, heads, dim)), np.zeros((t, heads)),
               np.zeros((t, heads, dim))]
        for b, n in enumerate(lengths):
            rows, m = slice(offsets[b], offsets[b + 1]), offsets[b + 1] - offsets[b]
            there = np.arange(min(n, table.shape[1] * self.bs))
            at, slot = table[b, there // self.bs], there % self.bs
            live = (at >= 0) & (at < self.blocks)
            at, slot = at[live], slot[live]
            if not m or not len(at):
                continue
            for h in range(self.heads):
                keys = dev(self.k[at, h, slot] * self.scale[at, h, 0, None])
                codes, y = dev(self.v[at, h, :, slot]), dev(self.scale[at, h, 1])
                vals = codes * y[:, None]
                f = slice(h * group, (h + 1) * group)
                x = dev(q[rows, f]).reshape(-1, dim)
                logits = x @ keys.t().contiguous() * scale
                lse = torch.logsumexp(logits, 1)
                p = torch.exp(logits - lse[:, None])
                g = (x.abs() @ keys.abs().t().contiguous() * abs(scale)).amax(1)
                least = (p * y).amax(1, keepdim=True) * codes.abs().sum(0)
                for o, z, tail in zip(out, (p @ vals, lse, p @ vals.abs(), g, least), ((dim,), (), (dim,), (), (dim,))):
                    o[rows, f] = z.view(m, group, *tail).cpu().numpy()
        return out


CHUNK, STEP = "k_chunk", "k_step"
FEW, ROWS, CROSS = "k_join_few", "k_join", "k_join_cross"

# kernel, waves of a workgroup, join of its splits: kv heads, group, dim, block tokens, type, rows, lengths, table's width
CASES = [
    (CHUNK, 4, None, 1, 16, 64, 16, F16, [19, 44, 172], [64, 0, 31], 4),
    (CHUNK, 4, None, 1, 16, 64, 64, BF16, [86, 176, 5], [256, 0, 130], 4),
    (CHUNK, 4, None, 1, 16, 96, 16, BF16, [39, 81, 150], [50, 64, 0], 4),
    (CHUNK, 4, None, 1, 16, 96, 64, F16, [86, 55, 139], [193, 0, 256], 4),
    (CHUNK, 4, None, 1, 8, 128, 16, BF16, [127, 295, 29], [61, 0, 64], 4),
    (CHUNK, 4, None, 1, 8, 128, 64, F16, [233, 11, 237], [251, 0, 256], 4),
    (CHUNK, 4, None, 1, 16, 192, 16, F16, [76, 140, 31], [64, 33, 0], 4),
    (CHUNK, 4, None, 1, 16, 192, 64, BF16, [213, 28, 27], [300, 0, 65], 5),
    (CHUNK, 4, None, 1, 16, 256, 16, BF16, [36, 104, 125], [0, 64, 47], 4),
    (CHUNK, 4, None, 1, 16, 256, 64, F16, [105, 9, 171], [200, 256, 0], 4),
    (CHUNK, 8, None, 8, 8, 64, 16, BF16, [15, 152, 83, 118, 81], [400, 0, 17, 399, 64], 25),
    (CHUNK, 8, None, 8, 8, 64, 64, F16, [151, 26, 7, 48, 248], [448, 0, 70, 448, 100], 7),
    (CHUNK, 4, FEW, 1, 16, 64, 16, BF16, [79, 170, 24], [464, 0, 250], 29),
    (CHUNK, 4, FEW, 1, 8, 64, 128, F16, [266, 157, 33], [512, 0, 385], 4),
    (CHUNK, 4, FEW, 1, 16, 96, 32, F16, [269, 3, 25], [416, 0, 200], 13),
    (CHUNK, 4, FEW, 1, 16, 96, 128, BF16, [206, 31, 10], [511, 0, 129], 4),
    (CHUNK, 4, FEW, 1, 16, 128, 16, F16, [237, 9, 38, 28], [460, 464, 0, 17], 29),
    (CHUNK, 4, FEW, 1, 8, 128, 64, BF16, [220, 158, 188], [448, 0, 129], 7),
    (CHUNK, 4, FEW, 1, 8, 192, 16, BF16, [65, 139, 272], [480, 0, 301], 30),
    (CHUNK, 4, FEW, 1, 16, 192, 128, F16, [23, 111, 123], [512, 300, 0], 4),
    (CHUNK, 4, FEW, 1, 16, 256, 16, F16, [79, 182, 34], [431, 0, 432], 27),
    (CHUNK, 4, FEW, 1, 16, 256, 64, BF16, [183, 34, 39], [447, 0, 65], 7),
    (CHUNK, 8, FEW, 4, 8, 64, 16, F16, [173, 64, 263], [1100, 0, 500], 73),
    (CHUNK, 8, FEW, 4, 2, 96, 128, F16, [85, 91, 265, 47], [3000, 0, 200, 3071], 24),
    (CHUNK, 8, FEW, 8, 1, 128, 32, F16, [30, 195, 200, 84, 40], [2368, 0, 700, 33, 1000], 74),
    (CHUNK, 8, FEW, 8, 3, 128, 64, BF16, [114, 15, 56, 34, 102], [1400, 0, 1472, 64, 65], 23),
    # 22 to 24 splits, which one lane walks
    (CHUNK, 4, FEW, 4, 3, 64, 64, BF16, [54, 76, 111, 30, 12], [300, 0, 64, 20000, 32300], 506),
    (CHUNK, 4, FEW, 2, 5, 96, 16, F16, [24, 36, 140, 47, 71], [14000, 0, 700, 100, 1], 876),
    (CHUNK, 8, FEW, 2, 8, 96, 32, BF16, [76, 11, 10, 20, 75], [100, 20000, 0, 19000, 31], 625),
    (CHUNK, 8, FEW, 2, 5, 128, 32, BF16, [290, 21, 39, 19], [400, 21500, 0, 20000], 674),
    (CHUNK, 4, FEW, 3, 4, 192, 32, BF16, [76, 103, 35, 38], [500, 0, 25000, 33], 782),
    (CHUNK, 4, FEW, 4, 2, 256, 32, F16, [138, 205, 11, 50, 4], [400, 0, 17400, 40, 9000], 545),
    (CHUNK, 4, ROWS, 1, 2, 128, 32, F16, [6, 52, 62], [31000, 0, 400], 970),
    (CHUNK, 4, ROWS, 1, 2, 256, 64, BF16, [7, 23, 37], [38000, 0, 100], 594),
    (CHUNK, 4, CROSS, 4, 3, 64, 16, F16, [34, 37, 4, 25], [500, 0, 11200, 11000], 700),
    (CHUNK, 8, CROSS, 1, 4, 64, 64, BF16, [18, 133, 191, 13], [12000, 0, 300, 12480], 195),
    (CHUNK, 4, CROSS, 1, 4, 96, 64, F16, [10, 115, 47, 208], [8000, 0, 8064, 65], 126),
    (CHUNK, 8, CROSS, 1, 4, 96, 32, BF16, [132, 113, 4], [5000, 0, 12700], 399),
    (CHUNK, 4, CROSS, 1, 2, 128, 32, BF16, [48, 93, 27, 7, 133], [6656, 0, 300, 6000, 33], 208),
    (CHUNK, 8, CROSS, 3, 8, 128, 64, F16, [58, 9, 14], [3000, 0, 3968], 62),
    (CHUNK, 4, CROSS, 2, 5, 192, 128, BF16, [10, 65, 32, 20], [8000, 0, 300, 8192], 64),
    (CHUNK, 4, CROSS, 2, 16, 256, 64, F16, [4, 8, 28], [3584, 0, 3000], 56),
    (STEP, 8, None, 1, 1, 64, 64, F16, [4, 11, 12], [832, 0, 65], 13),
    (STEP, 8, None, 3, 5, 96, 16, F16, [111, 8, 10], [300, 0, 1808], 113),
    (STEP, 8, None, 4, 2, 128, 16, BF16, [56, 25, 26, 121, 4], [2128, 0, 100, 5, 2000], 133),
    (STEP, 8, None, 8, 1, 192, 32, F16, [89, 66, 73], [2100, 0, 65], 66),
    (STEP, 8, None, 8, 3, 256, 64, BF16, [63, 12, 18, 4], [33, 0, 2752, 2700], 43),
    (STEP, 8, FEW, 1, 8, 96, 32, BF16, [34, 25, 32, 21, 64], [3616, 0, 3000, 1, 32], 113),
    (STEP, 8, FEW, 8, 1, 128, 32, F16, [40, 8, 26, 40, 4], [4704, 0, 100, 33, 4000], 147),
    (STEP, 8, FEW, 8, 1, 256, 64, F16, [40, 4, 30, 13], [100, 0, 65, 7800], 122),
    (STEP, 8, ROWS, 4, 1, 192, 16, BF16, [1, 12, 40], [18000, 0, 1000], 1145),
    (STEP, 4, CROSS, 1, 3, 192, 32, F16, [116], [11300], 354),
    (STEP, 4, CROSS, 1, 1, 256, 16, BF16, [159, 114, 31, 14], [400, 0, 20000, 15], 1309),
]


@pytest.mark.parametrize("case", CASES, ids=["%s-%s-%s-%dx%d-%d-%d-%s-%d" % (*c[:7], str(c[7])[6:], i) for i, c in enumerate(CASES)])
@pytest.mark.parametrize("holes,scale,aligned", [(0, None, True), (0.1, 0.3, False), (0, -0.1, True), (0.05, 0.0, False)])
def test_cross_attention_by_kernel(case, holes, scale, aligned):
    kernel, waves, join, heads, group, dim, bs, dt, news, lens, wide = case
    rng = np.random.default_rng(50)
    cache, table = shared(rng, heads, dim, bs, lens, 40, wide, holes, scale is None)
    off = offsets_of(news)
    q = queries(rng, off[-1], heads * group, dim, dt, aligned)
    scale = dim ** -0.5 if scale is None else scale
    t, n, o = dev(table), dev(np.int32(lens)), dev(off)

    def call():
        return kv.cross_attention(cache, q, t, n, o, scale=scale, max_tokens=max(news), return_lse=True)

    (got, lse), ran = launched(call)
    kind = f"{dim}, {flag(dt == BF16)}"
    mid = "false, " if kernel == STEP else ""
    assert ran == {f"{kernel}<{kind}, {mid}{flag(aligned)}, {waves}>"} | ({f"{join}<{kind}>"} if join else set())
    check(Whole(cache), got, lse, q, table, lens, off, scale)
    for a, b in zip(call(), (got, lse)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("at", [14, 26, 28, 36, 45, 52])
def test_graphs_of_each_kernel_replay(at):
    """Lengths, queries and places of the blocks change between replays; eager calls run between them."""
    kernel, waves, join, heads, group, dim, bs, dt, news, lens, wide = CASES[at]
    rng = np.random.default_rng(51)
    cache, table = shared(rng, heads, dim, bs, lens, 40, wide)
    q = queries(rng, sum(news), heads * group, dim, dt)
    t, n, o = dev(table), dev(np.int32(lens)), dev(offsets_of(news))

    def call():
        return kv.cross_attention(cache, q, t, n, o, max_tokens=max(news), return_lse=True)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(4):
        q.copy_(queries(rng, sum(news), heads * group, dim, dt))
        n.copy_(dev(np.int32(rng.permutation(lens))))
        t.copy_(dev(np.int32(rng.integers(-1, 42, table.shape))))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))
