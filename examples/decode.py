"""Decoding over a paged cache, dense and sparse: the attention operators as a program calls them.

    python examples/decode.py [--prompt 20000] [--steps 8] [--k 2048] [--packed]

Several sequences share a pool of pages. Their prompts' keys and values are appended in one call, the keys rotated on the
way. Every step then appends one token per sequence (its queries rotated in the same launch) and attends over the pages.
The longest sequence also keeps its rotated keys in a KeyCache, and attends to the exact top k of them: the sparse
attention, whose distance from the dense one is printed. With --packed the prompts are attended to as they come, in pieces, with
capped scores, and the steps attend over a second cache of 4-bit pages beside the first, whose distance is printed. Projections are
random: the point is the calls and their shapes.
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


def run_packed(prompt=20_000, steps=8, piece=4096, heads=32, kv_heads=8, head_dim=128, page=64, dtype=torch.bfloat16, cap=50.0, seed=0):
    """Prompts in pieces of `piece` tokens and then steps, over pages of dtype and of 4 bits. Returns the prompts' outputs and per
    step the queries and the outputs over both caches; both caches and what they were given."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    prompts = [prompt, prompt // 3, 1]
    rope = certex.Rotary(head_dim)
    most = -(-(prompt + steps) // page)
    pages = Pages(len(prompts) * most, page, most, len(prompts), kv_heads, head_dim, dtype)
    small = certex.PackedPages(len(prompts) * most, page, kv_heads, head_dim)
    outputs, given = [], []

    def step(counts):
        """counts[s] new tokens of every sequence into both caches; the rotated queries."""
        n = sum(counts)
        q, k, v = rand(n, heads, head_dim) * 4, rand(n, kv_heads, head_dim), rand(n, kv_heads, head_dim)
        before = list(pages.lengths)
        turned = pages.append(counts, k, v, rope, q=q)
        where = [(before[s] + i, s) for s, c in enumerate(counts) for i in range(c)]
        positions, owners = torch.tensor(where, dtype=torch.int32).cuda().T.contiguous()
        small.append(k, v, pages.table_gpu, positions, sequences=owners, rotary=rope)
        given.append((k, v, positions, owners))
        return turned

    left = list(prompts)
    while any(left):
        counts = [min(n, piece) for n in left]
        left = [n - c for n, c in zip(left, counts)]
        turned = step(counts)
        first = torch.tensor([sum(counts[:s]) for s in range(len(counts) + 1)], dtype=torch.int32).cuda()
        lengths = torch.tensor(pages.lengths, dtype=torch.int32).cuda()
        outputs.append((counts, turned, certex.prompt_attention(turned, pages.k, pages.v, pages.table_gpu, lengths, first, cap=cap)))
    results = []
    for _ in range(steps):
        turned = step([1] * len(prompts))
        lengths = torch.tensor(pages.lengths, dtype=torch.int32).cuda()
        dense = certex.paged_attention(turned, pages.k, pages.v, pages.table_gpu, lengths, cap=cap)
        results.append((turned, dense, small.attend(turned, pages.table_gpu, lengths, cap=cap)))
    return outputs, results, pages, small, given


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=20_000)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--k", type=int, default=2048)
    ap.add_argument("--packed", action="store_true")
    a = ap.parse_args()
    if a.packed:
        outputs, results, pages, small, _ = run_packed(a.prompt, a.steps)
        bytes_of = pages.k.nbytes + pages.v.nbytes
        print(f"{len(outputs)} pieces of prompts; 4-bit pages take {small.data.nbytes / bytes_of:.3f} of the others' memory")
        for i, (_, dense, packed) in enumerate(results):
            d, s = dense.float(), packed.float()
            print(f"step {i}: {pages.lengths[0] - a.steps + i + 1} positions: 4 bits from {dense.dtype} "
                  f"{float((s - d).norm() / d.norm()):.3f} of its norm")
        sys.exit(0)
    pages, cache, results = run(a.prompt, a.steps, a.k)
    for i, (dense, sparse) in enumerate(results):
        d, s = dense[0].float(), sparse.float()
        print(f"step {i}: {pages.lengths[0] - a.steps + i + 1} keys, top {cache.k}: sparse from dense "
              f"{float((s - d).norm() / d.norm()):.3f} of its norm")
