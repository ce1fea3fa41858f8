"""Attention of prompts and of bent scores against the float64 definition (shaped_reference.py)."""

import pytest
import torch

import libcertex_amd as certex
from tests import shaped_reference as ref
from tests.paged_reference import UNIT
from tests.test_paged_gpu import ints, paged, rand

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def weight_unit(dtype):
    """The weights of 16-bit types are rounded to the type."""
    return 0.0 if dtype == torch.float32 else UNIT[dtype]


def slopes_of(heads):
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)


def check_prompt(news, pasts, heads, kv, d, dv, page, dtype, window=None, prefix=None, cap=None, slopes=None, scale=None,
                 loud=1.0, seed=0, **kw):
    lens = [n + p for n, p in zip(news, pasts)]
    kp, vp, table, keys, values = paged(lens, page, kv, d, dv, dtype, seed=seed, **kw)
    first = [sum(news[:s]) for s in range(len(news) + 1)]
    q = rand(first[-1], heads, d, dtype=dtype, scale=loud, seed=seed + 1)
    how = dict(window=window, cap=cap, slopes=slopes, scale=scale, prefix=None if prefix is None else ints(prefix))
    out, lse = certex.prompt_attention(q, kp, vp, table, ints(lens), ints(first), return_lse=True, **how)
    assert out.shape == (first[-1], heads, dv) and out.dtype == dtype and lse.dtype == torch.float32
    for s, n in enumerate(lens):
        rows = slice(first[s], first[s + 1])
        want = ref.attend(q[rows], torch.arange(pasts[s], n), keys[s], values[s], d**-0.5 if scale is None else scale,
                          prefix=min(n, prefix[s]) if prefix else 0, window=window, cap=cap, slopes=slopes,
                          weight=weight_unit(dtype))
        ref.check(out[rows], lse[rows], want)
    wide = certex.prompt_attention(q, kp, vp, table, ints(lens, torch.int64), ints(first, torch.int64), **how)
    assert torch.equal(out, wide)  # runs repeat bit for bit
    return out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv", [(8, 2), (4, 4), (7, 1), (40, 2), (6, 2), (48, 1)])
def test_prompt_heads(gpu, dtype, heads, kv):
    check_prompt([1, 0, 33, 70, 129], [0, 5, 0, 64, 3], heads, kv, 64, 64, 16, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", [(128, 128), (96, 96), (80, 72), (256, 256), (192, 128), (64, 256), (8, 8), (33, 17),
                                   (130, 66), (1, 1), (128, 40), (255, 255), (3, 100)])
def test_prompt_dims(gpu, dtype, d, dv):
    check_prompt([5, 64, 100], [0, 31, 7], 4, 2, d, dv, 32, dtype, seed=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 1000])
@pytest.mark.parametrize("heads_first", [False, True])
def test_prompt_pages(gpu, dtype, page, heads_first):
    check_prompt([1, 7, 8, 9, 31, 64, 65, 130], [0, 1, 7, 64, 0, 63, 200, 9], 4, 2, 64, 64, page, dtype,
                 heads_first=heads_first, seed=4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 10_000])
def test_prompt_window(gpu, dtype, d, window):
    check_prompt([1, 0, 90, 200], [100, 3, 300, 0], 4, 2, d, d, 16, dtype, window=window, seed=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [None, 40])
def test_prompt_prefix(gpu, dtype, window):
    """Prefixes within the new tokens, over all of them, past the length, of nothing, and below the past."""
    check_prompt([130, 70, 40, 33, 90], [0, 0, 10, 5, 100], 6, 3, 64, 64, 16, dtype, prefix=[50, 70, 1000, 0, 60],
                 window=window, seed=6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap, lean", [(5.0, False), (50.0, False), (None, True), (30.0, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_bent(gpu, dtype, cap, lean, d):
    check_prompt([1, 90, 70], [200, 0, 33], 8, 2, d, d, 16, dtype, cap=cap, slopes=slopes_of(8) if lean else None, loud=4.0,
                 prefix=[0, 30, 5], seed=7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [65.0, 3e4, 1e6, 1e30])
def test_prompt_large_cap(gpu, dtype, cap):
    """A cap far beyond the scores leaves them: cap tanh(y / cap) is y within 5 units in the last place, with the y^3 / (3 cap^2)
    by which it is less."""
    lens, q = [200, 90], rand(60, 4, 64, dtype=dtype, seed=61)
    kp, vp, table, keys, values = paged(lens, 16, 2, 64, 64, dtype, seed=60)
    out, lse = certex.prompt_attention(q, kp, vp, table, ints(lens), ints([0, 20, 60]), cap=cap, return_lse=True)
    for s, rows in enumerate([slice(0, 20), slice(20, 60)]):
        n = rows.stop - rows.start
        scores = q[rows].double().cpu().abs().norm(dim=-1).max() * keys[s].double().cpu().norm(dim=-1).max() / 8
        bend = float(scores) ** 3 / (3 * cap**2) + 5 * 2.0**-24 * float(scores)
        want = ref.attend(q[rows], torch.arange(lens[s] - n, lens[s]), keys[s], values[s], 0.125, weight=weight_unit(dtype) + bend)
        if cap < 100:  # where the bend shows, the definition's own
            exact = ref.attend(q[rows], torch.arange(lens[s] - n, lens[s]), keys[s], values[s], 0.125, cap=cap)
            want = (*exact[:2], *want[2:])
        ref.check(out[rows], lse[rows], want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news, pasts", [([16], [20_000]), ([1, 1, 1, 2], [9_000, 50, 0, 3_000]), ([300], [2_000]),
                                         ([3] * 20, [100 * i for i in range(20)])])
def test_prompt_long(gpu, dtype, news, pasts):
    """Few tokens over long caches: their positions are split over workgroups and joined."""
    check_prompt(news, pasts, 8, 2, 128, 128, 64, dtype, seed=8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", [(256, 256), (256, 130), (40, 129 + 64), (201, 255), (160, 160), (161, 63), (9, 256)])
def test_prompt_wide_heads(gpu, dtype, d, dv):
    """Columns that two workgroups share, whole and split over positions, with logarithms of their own once."""
    check_prompt([20, 3], [1_500, 40], 4, 2, d, dv, 16, dtype, seed=62)
    check_prompt([200, 130, 1], [0, 9, 0], 3, 1, d, dv, 24, dtype, prefix=[50, 0, 0], cap=30.0, slopes=slopes_of(3), seed=63)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_extreme_scores(gpu, dtype):
    """Scores in the hundreds (one weight takes all), of a scale of 0 (all equal) and of a negative one."""
    for how in (dict(loud=30.0), dict(scale=0.0), dict(scale=-0.3), dict(scale=-0.3, cap=20.0, loud=4.0), dict(scale=0.0, cap=20.0)):
        check_prompt([100, 5], [30, 300], 4, 2, 128, 128, 16, dtype, seed=9, **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fill", [float("inf"), float("-inf"), 0.0])
def test_prompt_unused_slots(gpu, dtype, fill):
    """What slots past a length hold (NaN in the other tests) does not matter."""
    check_prompt([1, 40, 63, 65], [0, 0, 1, 100], 4, 2, 64, 64, 32, dtype, fill=fill, seed=10)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("past", [0, 70])
def test_prompt_unbounded_values(gpu, dtype, past):
    """An infinite or NaN key or value shows in the rows that see its position, and in no other row, column or head."""
    n, heads = 150, 4
    kp, vp, table, *_ = paged([past + n], 16, 2, 64, 64, dtype, seed=11)
    q = rand(n, heads, 64, dtype=dtype)
    lens, first = ints([past + n]), ints([0, n])
    clean = certex.prompt_attention(q, kp, vp, table, lens, first)
    for pos, value in ((past + 37, float("inf")), (past + 100, float("nan")), (past + 64, float("-inf")), (3, float("inf"))):
        at = int(table[0, pos // 16]), pos % 16
        keep = float(vp[at][1, 5])
        vp[at][1, 5] = value
        out = certex.prompt_attention(q, kp, vp, table, lens, first)
        vp[at][1, 5] = keep
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[max(0, pos - past) :, 2:, 5] = True
        assert not out[bad].isfinite().any() and torch.equal(out[~bad], clean[~bad])
        keep = kp[at].clone()
        kp[at][1, 5] = float("nan")
        out = certex.prompt_attention(q, kp, vp, table, lens, first)
        kp[at] = keep
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[max(0, pos - past) :, 2:] = True
        assert out[bad].isnan().all() and torch.equal(out[~bad], clean[~bad])
    q[20, 1] = float("nan")
    out, lse = certex.prompt_attention(q, kp, vp, table, lens, first, return_lse=True)
    assert out[20, 1].isnan().all() and lse[20, 1].isnan() and int(out.isnan().sum()) == 64


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_lowest_keys(gpu, dtype):
    """Keys of the type's lowest value drive scores to -inf or far down: those positions weigh nothing."""
    n = 70
    kp, vp, table, keys, values = paged([n], 16, 2, 64, 64, dtype, seed=12)
    for t in range(3, n):
        kp[int(table[0, t // 16]), t % 16] = torch.finfo(dtype).min
    q = torch.ones((n, 4, 64), dtype=dtype, device="cuda")
    out, lse = certex.prompt_attention(q, kp, vp, table, ints([n]), ints([0, n]), return_lse=True)
    there = torch.arange(n) < 3
    ref.check(out, lse, ref.attend(q, torch.arange(n), keys[0], values[0], 64**-0.5, there=there, weight=weight_unit(dtype)))


def test_prompt_lengths_and_holes(gpu):
    """Lengths below 0 and past the table, more tokens than positions, missing pages, tokens of no sequence."""
    dtype, page = torch.bfloat16, 16
    kp, vp, table, keys, values = paged([64] * 5, page, 2, 64, 64, dtype, seed=13)
    table[2, 1] = -1
    table[3] = ints([-1, 10_000, -5, kp.shape[0]])
    first = [3, 13, 33, 53, 60, 80]
    lens = [-3, 1_000_000, 64, 64, 12]
    q = rand(90, 4, 64, dtype=dtype)
    out, lse = certex.prompt_attention(q, kp, vp, table, ints(lens), ints(first), return_lse=True)
    empty = [*range(0, 13), *range(53, 60), *range(60, 68), *range(80, 90)]
    assert (out[empty] == 0).all() and (lse[empty] == float("-inf")).all()
    there = torch.arange(64) // page != 1
    unit = weight_unit(dtype)
    ref.check(out[13:33], lse[13:33], ref.attend(q[13:33], torch.arange(44, 64), keys[1], values[1], 64**-0.5, weight=unit))
    ref.check(out[33:53], lse[33:53],
              ref.attend(q[33:53], torch.arange(44, 64), keys[2], values[2], 64**-0.5, there=there, weight=unit))
    ref.check(out[68:80], lse[68:80], ref.attend(q[68:80], torch.arange(12), keys[4][:12], values[4][:12], 64**-0.5, weight=unit))
    none = certex.prompt_attention(q[:0], kp, vp, table, ints([64] * 5), ints([0] * 6))
    assert none.shape == (0, 4, 64)
    nobody, lse = certex.prompt_attention(q, kp, vp, table, ints([64] * 5), ints([0] * 6), return_lse=True)
    assert (nobody == 0).all() and (lse == float("-inf")).all()
    alone = certex.prompt_attention(q, kp, vp, table[:0], ints([]), ints([0]))
    assert (alone == 0).all()


def test_prompt_first_that_falls(gpu):
    """Offsets that fall or leave the tokens read and write nothing outside (the outputs of such a call are any)."""
    kp, vp, table, *_ = paged([64] * 4, 16, 2, 64, 64, torch.bfloat16, seed=14)
    q = rand(50, 4, 64, dtype=torch.bfloat16)
    for first in ([0, 30, 10, 40, 50], [-5, 100, 20, -7, 1 << 40], [50, 40, 30, 20, 10], [1 << 50] * 5):
        out = certex.prompt_attention(q, kp, vp, table, ints([64] * 4), ints(first, torch.int64))
        assert out.shape == q.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_unaligned(gpu, dtype):
    """Queries that are a slice of a projection (any alignment), pools with gaps between heads."""
    lens, news = [60, 200], [60, 90]
    kp, vp, table, keys, values = paged(lens, 16, 2, 64, 64, dtype, seed=15)
    wide = rand(150, 4, 200, dtype=dtype)
    both = torch.full((*kp.shape[:3], 131), float("nan"), dtype=dtype, device="cuda")
    both[..., 3:67], both[..., 67:] = kp, vp
    for q, k, v in [(wide[..., 1:65], kp, vp), (wide[..., 8:72], both[..., 3:67], both[..., 67:]),
                    (wide[..., ::3][..., :64], kp, both[..., 67:]), (wide.transpose(0, 1).contiguous().transpose(0, 1)[..., 5:69], kp, vp)]:
        out = certex.prompt_attention(q, k, v, table, ints(lens), ints([0, 60, 150]))
        for s, rows in enumerate((slice(0, 60), slice(60, 150))):
            want = ref.attend(q[rows], torch.arange(lens[s] - news[s], lens[s]), keys[s], values[s], 64**-0.5,
                              weight=weight_unit(dtype))
            ref.check(out[rows], None, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_many_sequences(gpu, dtype):
    """More sequences than a wave has lanes, most of them of one token or none."""
    g = torch.Generator().manual_seed(16)
    news = torch.randint(0, 4, (300,), generator=g).tolist()
    check_prompt(news, [i % 40 for i in range(300)], 2, 1, 64, 64, 16, dtype, seed=16)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_is_paged_attention_of_one_token(gpu, dtype):
    """One new token of every sequence: both operators' outputs are within their bounds of the same definition."""
    lens = [1, 90, 700, 2500]
    slopes = slopes_of(8)
    kp, vp, table, keys, values = paged(lens, 16, 2, 64, 64, dtype, seed=17)
    q = rand(4, 8, 64, dtype=dtype, scale=3.0)
    for how in (dict(), dict(cap=20.0), dict(slopes=slopes), dict(window=300, cap=20.0, slopes=slopes)):
        many, many_lse = certex.prompt_attention(q, kp, vp, table, ints(lens), ints([0, 1, 2, 3, 4]), return_lse=True, **how)
        one, one_lse = certex.paged_attention(q, kp, vp, table, ints(lens), return_lse=True, **how)
        for s, n in enumerate(lens):
            for out, lse, weight in ((many, many_lse, weight_unit(dtype)), (one, one_lse, 0.0)):
                ref.check(out[s : s + 1], lse[s : s + 1],
                          ref.attend(q[s : s + 1], torch.tensor([n - 1]), keys[s], values[s], 64**-0.5, weight=weight, **how))


# ---- one new token, bent scores ----


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", [(128, 128), (64, 64), (96, 96), (80, 72), (256, 256), (33, 17), (5, 3)])
@pytest.mark.parametrize("cap, lean, window", [(5.0, False, None), (50.0, True, 90), (None, True, None)])
def test_attend_bent(gpu, dtype, d, dv, cap, lean, window):
    lens = [1, 0, 33, 130, 700]
    slopes = slopes_of(8) if lean else None
    kp, vp, table, keys, values = paged(lens, 16, 2, d, dv, dtype, seed=18)
    q = rand(5, 8, d, dtype=dtype, scale=4.0)
    out, lse = certex.paged_attention(q, kp, vp, table, ints(lens), return_lse=True, cap=cap, slopes=slopes, window=window)
    for s, n in enumerate(lens):
        ref.check(out[s : s + 1], lse[s : s + 1], ref.attend(q[s : s + 1], torch.tensor([n - 1]), keys[s], values[s], d**-0.5,
                                                            cap=cap, slopes=slopes, window=window))


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_bent_long(gpu, dtype):
    """Sequences that shares cut; slopes of both signs; a slope of 0 and a cap that nothing reaches change little."""
    lens, heads = [20_000, 3, 4_000], 24
    kp, vp, table, keys, values = paged(lens, 64, 1, 64, 64, dtype, seed=19)
    q = rand(3, heads, 64, dtype=dtype)
    slopes = slopes_of(heads) * torch.where(torch.arange(heads, device="cuda") % 5 == 4, -0.01, 1.0)
    out, lse = certex.paged_attention(q, kp, vp, table, ints(lens), return_lse=True, slopes=slopes, cap=30.0)
    for s, n in enumerate(lens):
        ref.check(out[s : s + 1], lse[s : s + 1], ref.attend(q[s : s + 1], torch.tensor([n - 1]), keys[s], values[s], 64**-0.5,
                                                            cap=30.0, slopes=slopes))
    zero = certex.paged_attention(q, kp, vp, table, ints(lens), slopes=torch.zeros(heads, device="cuda"))
    for s, n in enumerate(lens):
        ref.check(zero[s : s + 1], None, ref.attend(q[s : s + 1], torch.tensor([n - 1]), keys[s], values[s], 64**-0.5))


def test_attend_bent_nan_is_seen(gpu):
    """A NaN key is not swallowed by the cap."""
    kp, vp, table, *_ = paged([50, 50], 16, 2, 64, 64, torch.bfloat16, seed=20)
    kp[int(table[0, 1]), 3, 1, 5] = float("nan")
    out = certex.paged_attention(rand(2, 4, 64, dtype=torch.bfloat16), kp, vp, table, ints([50, 50]), cap=10.0)
    assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and not out[1].isnan().any()


# ---- refusals ----


def test_refusals(gpu):
    kp, vp, table, *_ = paged([64] * 2, 16, 2, 64, 64, torch.bfloat16, seed=21)
    q = rand(10, 4, 64, dtype=torch.bfloat16)
    lens, first = ints([64, 64]), ints([0, 5, 10])

    def prompt(q=q, kp=kp, vp=vp, table=table, lens=lens, first=first, **kw):
        return certex.prompt_attention(q, kp, vp, table, lens, first, **kw)

    prompt()
    slopes = slopes_of(4)
    for kw, match in [
        (dict(first=ints([0, 10])), "first must have shape"), (dict(lens=ints([64])), "lengths must have shape"),
        (dict(prefix=ints([1])), "prefix must have shape"), (dict(cap=0.0), "positive"), (dict(cap=-1.0), "positive"),
        (dict(cap=float("nan")), "positive"), (dict(cap=float("inf")), "positive"), (dict(cap=1e-60), "positive"),
        (dict(cap=1e31), "too large"), (dict(cap=1e10, scale=1e-30), "too large"),
        (dict(window=0), "at least 1"),
        (dict(slopes=slopes[:3]), "slopes must have shape"), (dict(slopes=slopes.half()), "float32"),
        (dict(slopes=slopes.cpu()), "GPU"), (dict(scale=float("inf")), "finite"),
        (dict(q=q.float()), "as the other tensors"), (dict(q=q[:, :3]), "multiple of the key heads"),
        (dict(q=q[..., :32]), "same head dimension"), (dict(table=table[:1]), "lengths must have shape"),
        (dict(first=first.float()), "int32 or torch.int64"), (dict(q=q.cpu()), "GPU"),
        (dict(q=q.clone().requires_grad_()), "no gradient"), (dict(slopes=slopes.clone().requires_grad_()), "no gradient"),
    ]:
        with pytest.raises(ValueError, match=match):
            prompt(**kw)
    one = rand(2, 4, 64, dtype=torch.bfloat16)
    for kw, match in [(dict(cap=0.0), "positive"), (dict(slopes=slopes[:2]), "slopes must have shape"),
                      (dict(slopes=slopes.double()), "float32")]:
        with pytest.raises(ValueError, match=match):
            certex.paged_attention(one, kp, vp, table, lens, **kw)


# ---- streams and graphs ----


def test_prompt_in_a_graph(gpu):
    """Captured once and replayed over changed tokens, lengths and offsets, with eager calls between, also of two graphs that
    share a memory pool; split and whole tiles."""
    dtype = torch.bfloat16
    kp, vp, table, keys, values = paged([3000, 500], 16, 2, 64, 64, dtype, seed=22)
    q = rand(64, 4, 64, dtype=dtype)
    lens, first = ints([3000, 500]), ints([0, 30, 64])
    certex.prompt_attention(q, kp, vp, table, lens, first)
    graphs, outs = [], []
    for how in (dict(), dict(cap=20.0, slopes=slopes_of(4))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(certex.prompt_attention(q, kp, vp, table, lens, first, **how))
        graphs.append(g)
    for i, (ls, fs) in enumerate([([3000, 500], [0, 30, 64]), ([64, 500], [0, 64, 64]), ([2000, 31], [10, 33, 60])]):
        q.copy_(rand(64, 4, 64, dtype=dtype, seed=i))
        lens.copy_(ints(ls))
        first.copy_(ints(fs))
        for g, out, how in zip(graphs, outs, (dict(), dict(cap=20.0, slopes=slopes_of(4)))):
            g.replay()
            got = out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, certex.prompt_attention(q, kp, vp, table, lens, first, **how))


def test_prompt_on_a_stream(gpu):
    dtype = torch.float16
    kp, vp, table, *_ = paged([2000], 16, 2, 64, 64, dtype, seed=23)
    q = rand(40, 4, 64, dtype=dtype)
    want = certex.prompt_attention(q, kp, vp, table, ints([2000]), ints([0, 40]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [certex.prompt_attention(q, kp, vp, table, ints([2000]), ints([0, 40])) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(want, x) for x in got)
