"""The attention operators in a run, as a program calls them one after the other; and how precise the 4-bit attention is inside."""

import importlib.util
import os

import pytest
import torch

import libcertex_amd as certex
from tests import packed_reference as pack
from tests import shaped_reference as ref
from tests.paged_reference import UNIT
from tests.test_packed_gpu import packed, weight_unit
from tests.test_paged_gpu import ints, paged, rand

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode.py")


def test_packed_example(gpu):
    """Prompts in pieces, then steps, over 16-bit and 4-bit pages: every output against the definition, from the keys and values
    that were appended."""
    spec = importlib.util.spec_from_file_location("decode_example", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    heads, kv, d, cap = 8, 2, 64, 20.0
    outputs, results, pages, small, given = example.run_packed(prompt=300, steps=3, piece=128, heads=heads, kv_heads=kv, head_dim=d,
                                                               page=16, cap=cap)
    assert pages.lengths == [303, 103, 4] and len(outputs) == 3 and len(results) == 3
    rope = certex.Rotary(d)
    keys = [torch.empty(n, kv, d, dtype=torch.bfloat16, device="cuda") for n in pages.lengths]
    values = [torch.empty_like(x) for x in keys]
    for k, v, positions, owners in given:
        turned = rope(k, positions)
        for s in range(3):
            keys[s][positions[owners == s].long()], values[s][positions[owners == s].long()] = turned[owners == s], v[owners == s]
    half = UNIT[torch.bfloat16]
    seen = [0, 0, 0]
    for counts, q, out in outputs:
        at = 0
        for s, c in enumerate(counts):
            want = ref.attend(q[at : at + c], torch.arange(seen[s], seen[s] + c), keys[s][: seen[s] + c], values[s][: seen[s] + c],
                              d**-0.5, cap=cap, weight=half)
            ref.check(out[at : at + c], None, want)
            at, seen[s] = at + c, seen[s] + c
    for q, dense, quarter in results:
        for s in range(3):
            seen[s] += 1
            n = seen[s]
            k, v = keys[s][:n], values[s][:n]
            ref.check(dense[s : s + 1], None, ref.attend(q[s : s + 1], torch.tensor([n - 1]), k, v, d**-0.5, cap=cap))
            (held_k, k_sizes), (held_v, v_sizes) = pack.stored(k), pack.stored(v)
            ref.check(quarter[s : s + 1], None,
                      ref.attend(q[s : s + 1], torch.tensor([n - 1]), held_k, held_v, d**-0.5, cap=cap, key_sizes=k_sizes,
                                 value_sizes=v_sizes, weight=weight_unit(torch.bfloat16)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_are_the_prompt(gpu, dtype):
    """A prompt in pieces gives what it gives at once, within both calls' bounds."""
    n, heads = 500, 4
    kp, vp, table, keys, values = paged([n], 16, 2, 64, 64, dtype, seed=30)
    q = rand(n, heads, 64, dtype=dtype)
    want = ref.attend(q, torch.arange(n), keys[0], values[0], 64**-0.5, weight=0.0 if dtype == torch.float32 else UNIT[dtype])
    whole, lse = certex.prompt_attention(q, kp, vp, table, ints([n]), ints([0, n]), return_lse=True)
    ref.check(whole, lse, want)
    at = 0
    for c in (1, 64, 130, 5, 300):
        out = certex.prompt_attention(q[at : at + c], kp, vp, table, ints([at + c]), ints([0, c]))
        ref.check(out, None, tuple(x[at : at + c] for x in want))
        at += c


@pytest.mark.parametrize("tokens", [1, 10, 40])
def test_tokens_of_no_sequence(gpu, tokens):
    kp, vp, table, *_ = paged([64], 16, 2, 64, 64, torch.bfloat16, seed=31)
    q = rand(tokens, 4, 64, dtype=torch.bfloat16)
    out, lse = certex.prompt_attention(q, kp, vp, table[:0], ints([]), ints([0]), return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()


def test_pools_without_pages(gpu):
    """Empty pools and page tables: zeros."""
    q = rand(3, 4, 64, dtype=torch.bfloat16)
    none = torch.empty((0, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    assert (certex.prompt_attention(q, none, none, table, ints([5, 5, 5]), ints([0, 1, 2, 3])) == 0).all()
    empty = certex.PackedPages(0, 16, 2, 64)
    assert (empty.attend(q, table, ints([5, 5, 5])) == 0).all()
    empty.append(q[:, :2], q[:, :2], table, ints([0, 1, 2]))
    assert (empty.read(table, ints([0, 1, 2]))[0] == 0).all()
    assert (empty.attend(q, table[:, :0], ints([5, 5, 5])) == 0).all()


def test_cap_too_small_for_the_scale(gpu):
    kp, vp, table, *_ = paged([64], 16, 2, 64, 64, torch.bfloat16, seed=32)
    q = rand(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="too small"):
        certex.paged_attention(q, kp, vp, table, ints([64]), cap=1e-38)
    with pytest.raises(ValueError, match="too small"):
        certex.prompt_attention(q, kp, vp, table, ints([64]), ints([0, 1]), cap=1e-38)


@pytest.mark.parametrize("n", [4096, 65_536, 131_072])
def test_packed_float32_does_not_drift(gpu, n):
    """Single precision over long caches: sums over codes and over offsets do not grow beside the output. As random roundings an
    output is off by the errors of its weights, whose square sum its norm has too: e of a weight, 4 (sqrt(d) + 4) u sum |q k| / sqrt(d)
    in the mean over dimensions, and 8 u of the exponential, the weight, its two elements and the sums; 4 times that is the bound."""
    d, kv, heads = 128, 1, 4
    pages = certex.PackedPages(n // 64, 64, kv, d)
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda")[None]
    k, v = rand(n, kv, d, seed=33), rand(n, kv, d, seed=34)
    k[..., ::32] *= 4
    positions = torch.arange(n, device="cuda")
    pages.append(k, v, table, positions, sequences=torch.zeros_like(positions))
    q = rand(1, heads, d, seed=35)
    out, lse = pages.attend(q, table, ints([n]), return_lse=True)
    held_k, held_v = (x[:, 0].double() for x in pages.read(table, positions, sequences=torch.zeros_like(positions), dtype=torch.float32))
    s = q[0].double() @ held_k.T * d**-0.5
    w = torch.softmax(s, -1)
    want = w @ held_v
    size = float(((q[0].double().abs() @ held_k.abs().T) * d**-0.5).mean())
    u = 2.0**-24
    assert float((out[0].double() - want).norm() / want.norm()) <= 4 * (size / d**0.5 + 8) * u
    assert float((lse[0].double() - torch.logsumexp(s, -1)).abs().max()) <= 4 * (size / d**0.5 + 8) * u + 8 * u * float(lse.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_two_streams_at_once(gpu, dtype):
    """Calls of two streams, each with workspaces of its own, beside each other."""
    kp, vp, table, *_ = paged([5000, 300], 16, 2, 64, 64, dtype, seed=36)
    pages, small_table, *_ = packed([5000, 300], 16, 2, 64, 64, dtype, seed=36)
    q, many = rand(2, 8, 64, dtype=dtype), rand(40, 8, 64, dtype=dtype, seed=1)
    lens, first = ints([5000, 300]), ints([0, 15, 40])

    def calls():
        return (certex.prompt_attention(many, kp, vp, table, lens, first), certex.paged_attention(q, kp, vp, table, lens, cap=9.0),
                pages.attend(q, small_table, lens))

    want = calls()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(calls())
    for s in streams:
        s.synchronize()
    assert all(torch.equal(x, y) for outs in got for x, y in zip(outs, want))
