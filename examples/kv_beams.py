"""Beam decoding over a key-value cache whose blocks have owners: the prompts of several
users fork into beams, which share the prompt's blocks; at every step beams are
chosen anew, get room for a token, copy the blocks that they are about to write and still share, and attend in two parts,
the prompt's whole blocks once for all beams of a user and each beam's own tokens,
which are joined. At the end one beam of each user goes on with every second token, in blocks of its own.

    python examples/kv_beams.py [--users 8 --beams 8 --prompt 20000 --steps 64 --layers 4]

Prints, for every few steps, the blocks that are owned and those that the beams would own if they shared none, how far the
joined attention is from the one over all of a beam's tokens, and the time of both. Queries, keys
and scores are synthetic.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from dance_amd import kv  # noqa: E402


def run(users=8, beams=8, prompt=20000, steps=64, layers=4, heads=32, kv_heads=8, dim=128, block_tokens=64, seed=1, quiet=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def noise(*shape):
        return torch.randn(shape, generator=g, device="cuda").bfloat16()

    def ints(x):
        return torch.as_tensor(x, device="cuda").int()

    rows = users * beams
    prompts = [max(1, prompt - 331 * u) for u in range(users)]
    width = -(-(max(prompts) + steps) // block_tokens)
    # the prompts once, each beam's own tokens, and room for half of one beam each at the end
    each = steps // block_tokens + 3
    blocks = sum(-(-n // block_tokens) for n in prompts) * 3 // 2 + (rows + users) * each
    caches = [kv.KVCache.empty(blocks, kv_heads, dim, block_tokens) for _ in range(layers)]
    pages = kv.Pages.empty(blocks, block_tokens)

    # the prompts, then as many beams of each
    table, lengths = torch.full((users, width), -1, dtype=torch.int32, device="cuda"), ints([0] * users)
    now, _, _ = kv.reserve(pages, table, lengths, ints(prompts))
    assert now.tolist() == prompts, "the pool has no room for the prompts"
    offsets = ints([0] + prompts).cumsum(0).int()
    for cache in caches:
        kv.append(cache, noise(sum(prompts), kv_heads, dim), noise(sum(prompts), kv_heads, dim), table, now, offsets)
    table, lengths = kv.fork(pages, table, lengths, ints([u for u in range(users) for _ in range(beams)]))

    # whole blocks of the prompts, which no beam ever writes
    whole = [n // block_tokens for n in prompts]
    shared, shared_lengths = table[::beams, :max(1, max(whole))].contiguous(), ints([n * block_tokens for n in whole])
    groups = ints(range(0, rows + 1, beams))
    skip = ints([n for n in whole for _ in range(beams)])
    most = max(-(-(n + steps) // block_tokens) - w for n, w in zip(prompts, whole))
    places = skip[:, None] + torch.arange(most, device="cuda")
    places, inside = places.clamp(max=width - 1).long(), places < width

    out = []
    for step in range(steps):
        # beams that go on, each user's own
        parents = torch.randint(0, beams, (users, beams), generator=g, device="cuda")
        parents += torch.arange(users, device="cuda")[:, None] * beams
        table, lengths = kv.fork(pages, table, lengths, parents.view(-1).int() if step else ints(range(rows)))
        now, src, dst = kv.reserve(pages, table, lengths, lengths + 1)
        kv.copy(caches, src, dst)
        own = torch.where(inside, table.gather(1, places), -1)
        marks = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        apart = torch.zeros((), device="cuda")
        spent = [0.0, 0.0]
        for cache in caches:
            q = noise(rows, heads, dim)
            kv.append(cache, noise(rows, kv_heads, dim), noise(rows, kv_heads, dim), table, now)
            marks[0].record()
            a, l = kv.cross_attention(cache, q, shared, shared_lengths, groups, max_tokens=beams, return_lse=True)
            b, m = kv.attention(cache, q, own, now - skip * block_tokens, return_lse=True)
            joined = kv.join([a, b], [l, m])
            marks[1].record()
            full = kv.attention(cache, q, table, now)
            marks[2].record()
            apart = torch.maximum(apart, (joined.float() - full.float()).norm() / full.float().norm())
            torch.cuda.synchronize()
            spent = [s + 1e3 * x.elapsed_time(y) for s, x, y in zip(spent, marks, marks[1:])]
        out.append({"step": step, "owned": int((pages.refs > 0).sum()), "named": int((table >= 0).sum()), "apart": float(apart),
                    "missed": int((now == 0).sum()), "joined_us": spent[0] / layers, "full_us": spent[1] / layers})
        if not quiet and (step % 16 == 0 or step == steps - 1):
            print("step %3d: %d blocks for %d that the beams name, outputs differ by %.4f; in two parts %.0f us a layer, "
                  "in one %.0f us" % tuple(out[-1][k] for k in ("step", "owned", "named", "apart", "joined_us", "full_us")))

    # the first beam of each user, every second token of it; then nobody owns the rest
    table, lengths = kv.fork(pages, table, lengths, ints(range(0, rows, beams)))
    counts = (lengths + 1) // 2
    kept = torch.full_like(table, -1)
    room, _, _ = kv.reserve(pages, kept, torch.zeros_like(lengths), counts)
    keep = (2 * torch.arange(int(counts.max()), device="cuda")).int().expand(users, 1, -1).contiguous()
    for cache in caches:
        kv.compact(cache, keep, room, table, lengths, kept)
    kv.release(pages, table, lengths, keep=torch.zeros_like(lengths))
    q = noise(users, heads, dim)
    a = kv.attention(caches[0], q, kept, room)
    out[-1]["left"] = int((pages.refs > 0).sum())
    assert room.tolist() == counts.tolist() and bool(torch.isfinite(a).all())
    if not quiet:
        print("every second token of one beam each: %d blocks" % out[-1]["left"])
    return out


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("users", 8), ("beams", 8), ("prompt", 20000), ("steps", 64), ("layers", 4), ("seed", 1)):
        p.add_argument("--" + name, type=int, default=value)
    run(**vars(p.parse_args()))
