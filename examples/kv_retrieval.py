"""A decoding loop over a key-value cache in 8-bit codes: prompts of different
lengths enter the cache in chunks, then every step writes its tokens, selects the
blocks of the context worth reading, and attends to those.

    python examples/kv_retrieval.py [--seqs 8 --prompt 100000 --steps 32 --count 64]

Prints, for every few steps, the share of the full softmax's weight that the
selected blocks hold (exp of the difference of the two logarithms of the sums), the share of
as many newest blocks, how far the selection's outputs are from the full ones, and the time of a step with the selection and with all
of the context. Queries and keys are synthetic: a few directions that come back
through the context, as topics do in a text.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from dance_amd import kv  # noqa: E402


class Rows:
    """Synthetic keys, values and queries of one layer: a topic's direction and noise."""

    def __init__(self, heads, kv_heads, dim, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.topics = self.noise(32, kv_heads, dim)

    def noise(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def draw(self, tokens, topic):
        """Queries, keys and values of `tokens` tokens; topic: the topic of each."""
        t = self.topics[topic]
        k = 0.5 * t + self.noise(tokens, self.kv_heads, self.dim)
        q = t.repeat_interleave(self.heads // self.kv_heads, 1) + 0.5 * self.noise(tokens, self.heads, self.dim)
        v = self.noise(tokens, self.kv_heads, self.dim) + t
        return q.bfloat16(), k.bfloat16(), v.bfloat16()


def run(seqs=8, prompt=100000, steps=32, count=64, heads=32, kv_heads=8, dim=128, block_tokens=64, chunk=4096, seed=1,
        quiet=False):
    rows = Rows(heads, kv_heads, dim, seed)
    lengths = [max(1, prompt - 997 * b) for b in range(seqs)]
    per = -(-(max(lengths) + steps) // block_tokens)
    cache = kv.KVCache.empty(seqs * per, kv_heads, dim, block_tokens)
    table = torch.randperm(seqs * per, generator=rows.g, device="cuda").int().view(seqs, per)

    # the prompts, a chunk of every sequence at a time
    done = [0] * seqs
    while any(d < n for d, n in zip(done, lengths)):
        part = [min(chunk, n - d) for d, n in zip(done, lengths)]
        done = [d + p for d, p in zip(done, part)]
        offsets = torch.tensor([0] + part, device="cuda").cumsum(0).int()
        now = torch.tensor(done, dtype=torch.int32, device="cuda")
        # a topic lasts for a few hundred tokens
        topic = torch.randint(0, 32, (sum(part) // 256 + 1,), generator=rows.g, device="cuda").repeat_interleave(256)
        q, k, v = rows.draw(sum(part), topic[:sum(part)])
        kv.append(cache, k, v, table, now, offsets, max_tokens=max(part))
        kv.attention(cache, q, table, now, offsets, max_tokens=max(part))

    marks = [[torch.cuda.Event(enable_timing=True) for _ in range(3)] for _ in range(steps)]
    got = []
    now = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for step in range(steps):
        now += 1
        topic = torch.randint(0, 32, (seqs,), generator=rows.g, device="cuda")
        q, k, v = rows.draw(seqs, topic)
        kv.append(cache, k, v, table, now)
        marks[step][0].record()
        chosen = kv.select(cache, q, table, now, count, sink=1, recent=2)
        some, some_lse = kv.sparse_attention(cache, q, chosen, table, now, return_lse=True)
        marks[step][1].record()
        full, full_lse = kv.attention(cache, q, table, now, return_lse=True)
        marks[step][2].record()
        last = torch.arange(count, device="cuda") + ((now + block_tokens - 1) // block_tokens - count)[:, None]
        last = last.int()[:, None].expand(-1, kv_heads, -1).contiguous()  # negative where there are fewer
        _, last_lse = kv.sparse_attention(cache, q, last, table, now, return_lse=True)
        mass, newest = torch.exp(some_lse - full_lse).mean(), torch.exp(last_lse - full_lse).mean()
        apart = (some.float() - full.float()).norm() / full.float().norm()
        got.append((mass, newest, apart))
    torch.cuda.synchronize()
    out = []
    for step, (mass, newest, apart) in enumerate(got):
        a, b, c = marks[step]
        out.append({"step": step, "mass": float(mass), "newest": float(newest), "apart": float(apart),
                    "selected_us": 1e3 * a.elapsed_time(b),
                    "full_us": 1e3 * b.elapsed_time(c)})
        if not quiet and (step % 8 == 0 or step == steps - 1):
            print("step %3d: %d of about %d blocks hold %.3f of the weight (the newest %.3f), outputs differ by %.3f; "
                  "selected %.0f us, all %.0f us" % (step, count, max(lengths) // block_tokens, mass, newest, apart,
                                                     out[-1]["selected_us"], out[-1]["full_us"]))
    return out


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("seqs", 8), ("prompt", 100000), ("steps", 32), ("count", 64), ("seed", 1)):
        p.add_argument("--" + name, type=int, default=value)
    run(**vars(p.parse_args()))
