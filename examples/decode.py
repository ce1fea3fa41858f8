"""Decoding over a paged cache, dense and sparse: the attention operators as a program calls them.

    python examples/decode.py [--prompt 20000] [--steps 8] [--k 2048]

Several sequences share a pool of pages. Their prompts' keys and values are appended in one call, the keys rotated on the
way. Every step then appends one token per sequence (its queries rotated in the same launch) and attends over the pages.
The longest sequence also keeps its rotated keys in a KeyCache, and attends to the exact top k of them: the sparse
attention, whose distance from the dense one is printed. Projections are random: the point is the calls and their shapes.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import libcertex_amd as certex  # noqa: E402


class Pages:
    """A pool of pages for several sequences: which page holds what, on the host, and the table on the GPU."""

    def __init__(self, n_pages, page, max_pages, sequences, kv_heads, head_dim, dtype):
        self.page, self.free = page, list(range(n_pages))[::-1]
        self.lengths = [0] * sequences
        self.table = torch.full((sequences, max_pages), -1, dtype=torch.int32)  # the host's copy
        self.table_gpu = self.table.cuda()
        self.k = torch.empty((n_pages, page, kv_heads, head_dim), dtype=dtype, device="cuda")
        self.v = torch.empty_like(self.k)

    def append(self, counts, k, v, rope, q=None):
        """counts[s] new tokens of every sequence, in order; the rotated queries, if given."""
        positions, owners, grown = [], [], False
        for s, n in enumerate(counts):
            for p in range(self.lengths[s], self.lengths[s] + n):
                if p % self.page == 0:
                    self.table[s, p // self.page] = self.free.pop()
                    grown = True
                positions.append(p)
                owners.append(s)
            self.lengths[s] += n
        if grown:
            self.table_gpu.copy_(self.table)
        where = torch.tensor([positions, owners], dtype=torch.int32).cuda()
        return certex.append_pages(k, v, self.k, self.v, self.table_gpu, where[0], sequences=where[1], rotary=rope, q=q)

    def attend(self, q, window=None):
        return certex.paged_attention(q, self.k, self.v, self.table_gpu, torch.tensor(self.lengths, device="cuda"),
                                      window=window)


def run(prompt=20_000, steps=8, k=2048, heads=32, kv_heads=8, head_dim=128, page=64, dtype=torch.bfloat16, seed=0):
    """Per step: the dense outputs of every sequence, and the sparse ones of the first; both as the program has them."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    prompts = [prompt, prompt // 3, 1, prompt // 50]
    rope = certex.Rotary(head_dim, scaling="ramp", factor=4.0, original_length=max(256, prompt // 4))
    most = -(-(prompt + steps) // page)
    pages = Pages(len(prompts) * most, page, most, len(prompts), kv_heads, head_dim, dtype)
    keys, values = rand(sum(prompts), kv_heads, head_dim), rand(sum(prompts), kv_heads, head_dim)
    pages.append(prompts, keys, values, rope)
    # the longest sequence's keys, rotated, to the cache that finds the top k
    cache = certex.KeyCache(kv_heads, head_dim, k=min(k, prompt), capacity=prompt + steps)
    cache.append(rope(keys[:prompt], torch.arange(prompt, device="cuda")).transpose(0, 1))
    results = []
    for _ in range(steps):
        q, new_k, new_v = (rand(len(prompts), h, head_dim) for h in (heads, kv_heads, kv_heads))
        q *= 4  # as trained queries do, so that a few keys hold most of the weight
        turned = pages.append([1] * len(prompts), new_k, new_v, rope, q=q)
        dense = pages.attend(turned)
        last = torch.tensor([pages.lengths[0] - 1], device="cuda")
        cache.append(rope(new_k[:1], last).transpose(0, 1))
        sparse = cache.attend(turned[0], pages.v, page_table=pages.table_gpu[0])
        results.append((dense, sparse))
    return pages, cache, results


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=20_000)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--k", type=int, default=2048)
    a = ap.parse_args()
    pages, cache, results = run(a.prompt, a.steps, a.k)
    for i, (dense, sparse) in enumerate(results):
        d, s = dense[0].float(), sparse.float()
        print(f"step {i}: {pages.lengths[0] - a.steps + i + 1} keys, top {cache.k}: sparse from dense "
              f"{float((s - d).norm() / d.norm()):.3f} of its norm")
