"""The decoding example: its pages and outputs against the float64 definitions."""

import importlib.util
import os

import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode.py")


def test_decode_example(gpu):
    spec = importlib.util.spec_from_file_location("decode_example", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    prompt, steps, heads, kv, d = 600, 3, 8, 2, 64
    pages, cache, results = example.run(prompt=prompt, steps=steps, k=prompt, heads=heads, kv_heads=kv, head_dim=d, page=16)
    assert pages.lengths == [603, 203, 4, 15] and cache.size == 603 and len(results) == steps
    # the same random numbers again, through the definitions
    g = torch.Generator(device="cuda").manual_seed(0)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

    import libcertex_amd as certex

    rope = certex.Rotary(d, scaling="ramp", factor=4.0, original_length=256)
    prompts = [600, 200, 1, 12]
    k, v = rand(813, kv, d), rand(813, kv, d)
    first = [0, 600, 800, 801, 813]
    keys = [rope(k[a:b], torch.arange(b - a, device="cuda")) for a, b in zip(first, first[1:])]
    values = [v[a:b] for a, b in zip(first, first[1:])]
    for i, (dense, sparse) in enumerate(results):
        q, nk, nv = (rand(4, h, d) for h in (heads, kv, kv))
        pos = torch.tensor([n + i for n in prompts], device="cuda")
        q, nk = rope(q * 4, pos), rope(nk, pos)
        for s in range(4):
            keys[s], values[s] = torch.cat([keys[s], nk[s : s + 1]]), torch.cat([values[s], nv[s : s + 1]])
            want, _, spread, dots = ref.attend(q[s], keys[s], values[s], d**-0.5)
            ref.assert_attended(dense[s], want, spread, dots, len(keys[s]), d)
            if s == 0:  # the top 600 of 601 to 603 keys
                scores = (q[0].double().view(kv, heads // kv, d) @ keys[0].double().permute(1, 2, 0).contiguous()).cpu()
                kept, ids = scores.view(heads, -1).topk(prompt, -1)
                w = torch.softmax(kept * d**-0.5, -1)
                for h in range(heads):
                    rows = values[0][ids[h].cuda(), h // (heads // kv)].double().cpu()
                    ref.assert_attended(sparse[h][None], (w[h] @ rows)[None], (w[h] @ rows.abs())[None], dots[h : h + 1], prompt, d)
