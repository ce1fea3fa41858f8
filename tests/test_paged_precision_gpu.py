"""How precise the attention operators are inside, where the rounding of their outputs does not hide it: values that
cancel, scores far from 0. Bounds are in units u = 2^-24, half a unit in the last place of float32."""

import math

import pytest
import torch

import libcertex_amd as certex
from tests import paged_reference as ref
from tests.test_paged_gpu import paged

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0**-24


def cancelling(weights, width, dtype, seed):
    """Values (rows, n, width) of a type whose sums under the softmax weights (rows, n) leave little of their terms: each
    value cancels the sum of those before it as far as the type goes."""
    g = torch.Generator().manual_seed(seed)
    rows, n = weights.shape
    v = torch.zeros((rows, n, width), dtype=torch.float64)
    v[:, 0] = (256 * (1 + torch.rand((rows, width), generator=g, dtype=torch.float64))).to(dtype).double()
    left = weights[:, :1] * v[:, 0]
    for t in range(1, n):
        v[:, t] = (-left / weights[:, t : t + 1]).to(dtype).double()
        left = left + weights[:, t : t + 1] * v[:, t]
    return v


def check_cancelled(out, w, v, dtype, units):
    """|out - sum w v| <= units u sum w |v|, and the output's rounding: half a unit in its last place."""
    want, spread = (w[..., None] * v).sum(2), (w[..., None] * v.abs()).sum(2)
    bound = units * U * spread + (ref.UNIT[dtype] + units * U) * want.abs() + ref.UNIT[dtype] * torch.finfo(dtype).tiny
    assert (want.abs() < spread / 1000).all()  # that hides nothing
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() / bound).max())


def attend_scores(s, v, dtype, scale, base=0.0):
    """paged_attention over exact scores base + s (rows, heads, n) and values v (rows, heads, n, d); float64."""
    b, h, n, d = v.shape
    kp, vp = torch.zeros((b, 8, h, d), dtype=dtype), torch.zeros((b, 8, h, d), dtype=dtype)
    kp[:, :n, :, 0], kp[:, :n, :, 1] = s.transpose(1, 2).to(dtype), base
    vp[:, :n] = v.transpose(1, 2).to(dtype)
    q = torch.zeros((b, h, d), dtype=dtype)
    q[..., :2] = 1.0
    assert torch.equal(kp[:, :n, :, 0].double(), s.transpose(1, 2).double()) and (kp[:, :n, :, 1] == base).all()
    assert torch.equal(vp[:, :n].double(), v.transpose(1, 2))
    table = torch.arange(b, dtype=torch.int32).view(b, 1)
    return certex.paged_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.full((b,), n, device="cuda"),
                                  scale=scale).double().cpu()


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_weights_are_whole(gpu, dtype):
    """The softmax's weights enter the product with the values as float32 has them. Scores are exact, |scale score| <= 1:
    a weight is off by 5 u of its exponent (|x| <= 1.5 and differences to 2.9 in powers of 2, rounded three times), 2 u of
    the exponential and u of its own; 8 u are for the sums."""
    b, h, d, n = 32, 4, 64, 4
    g = torch.Generator().manual_seed(1)
    s = torch.randint(-128, 129, (b, h, n), generator=g) / 128.0
    w = torch.softmax(s.double(), -1)
    v = cancelling(w.reshape(b * h, n), d, dtype, 2).reshape(b, h, n, d)
    check_cancelled(attend_scores(s, v, dtype, 1.0), w, v, dtype, 16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("base", [0, 344 - 8, 2752, 32768])
def test_attend_scores_far_from_zero(gpu, dtype, base):
    """A score's exponent is rounded after the maximum has left it. Scores are exact and differ by up to D = 6.5 in powers
    of 2: the scale's rounding and their product's take u D ln 2 each, 9 u; 3 u are the exponential's and the weight's, 8 u
    the sums'. (At a score of 344.85 or 2758.8, a scale of 0.75 times log2(e) is half a unit in the last place off.)"""
    b, h, d, n = 32, 4, 64, 4
    g = torch.Generator().manual_seed(5)
    s = 4 + torch.randint(0, 48, (b, h, n), generator=g) / 8.0
    w = torch.softmax(0.75 * s.double(), -1)
    v = cancelling(w.reshape(b * h, n), d, dtype, 6).reshape(b, h, n, d)
    check_cancelled(attend_scores(s, v, dtype, 0.75, base), w, v, dtype, 20)


# few queries a head gather rows; many, over values larger than a die's cache, go by ranges
ROUTES = [(2, 500, 300, 4), (64, 40_000, 2050, 128)]


@pytest.mark.parametrize("queries, n, k, width", ROUTES)
@pytest.mark.parametrize("offset", [0.0, 200.0, 5000.0, 1e6, -1e6])
def test_selected_scores_far_from_zero(gpu, queries, n, k, width, offset):
    """Scores are exact inputs, so that an offset that all of them share rounds nothing: what is rounded is their distances,
    of up to D = 12 in powers of 2, three times (3 u D ln 2 = 25 u), besides 3 u of the exponential and the weight; each
    of the two sums of k terms takes 4 sqrt(k) u."""
    heads, kv, scale = 4, 2, 0.25
    g = torch.Generator(device="cuda").manual_seed(3)
    spread = torch.randint(0, 8 * 33, (heads, queries, k), generator=g, device="cuda") / 8.0  # scale * 33 * log2(e) < 12
    scores, ids = spread + offset, torch.randint(0, n, (heads, queries, k), generator=g, device="cuda")
    assert torch.equal(scores.double() - offset, spread.double())
    values = torch.randn((kv, n, width), generator=g, device="cuda")
    out, lse = certex.selected_attention(scores, ids, values, scale, return_lse=True)
    host = values.double().cpu()
    for h in range(heads):
        for i in range(0, queries, 7):
            w = torch.softmax(scale * scores[h, i].double().cpu(), 0)
            rows = host[h // 2, ids[h, i].cpu()]
            size = (w @ rows.abs()).norm()
            e = (28 + 8 * k**0.5) * U
            assert float((out[h, i].double().cpu() - w @ rows).norm() / size) <= e
            want = torch.logsumexp(scale * scores[h, i].double().cpu(), 0)
            assert abs(float(lse[h, i].double().cpu() - want)) <= e + 4 * U * abs(float(want))


@pytest.mark.parametrize("queries, n, k, width", ROUTES)
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.0])
def test_selected_lowest_scores(gpu, queries, n, k, width, scale):
    """Scores of float32's lowest value, which masks are made of: they weigh nothing next to others, and alike where a row
    holds no other, whose scaled scores are as finite; with a scale of 0 all weigh alike."""
    low = torch.finfo(torch.float32).min if scale >= 0 else torch.finfo(torch.float32).max
    g = torch.Generator(device="cuda").manual_seed(4)
    scores = torch.randn((4, queries, k), generator=g, device="cuda")
    ids = torch.randint(0, n, (4, queries, k), generator=g, device="cuda")
    scores[:2] = low
    scores[2:, :, k // 3 :] = low
    scores[3, 1, 7] = -low  # as far from the others as scores can be
    values = torch.randn((2, n, width), generator=g, device="cuda")
    out, lse = certex.selected_attention(scores, ids, values, scale, return_lse=True)
    host = values.double().cpu()
    for h in range(4):
        for i in {0, 1, queries - 1}:
            s = scale * scores[h, i].double().cpu()
            w, rows = torch.softmax(s, 0), host[h // 2, ids[h, i].cpu()]
            e = (28 + 8 * k**0.5) * U
            assert float((out[h, i].double().cpu() - w @ rows).norm() / (w @ rows.abs()).norm()) <= e
            want = torch.logsumexp(s, 0)
            assert abs(float(lse[h, i].double().cpu() - want)) <= e + 4 * U * abs(float(want))


@pytest.mark.parametrize("queries, n, k, width", ROUTES)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("last", [False, True])
def test_selected_value_of_a_vanishing_weight(gpu, queries, n, k, width, value, last):
    """A selected value that is not finite shows in its column even where its weight is too small for float32, whichever
    way the ids are taken; a score of -inf keeps it out."""
    g = torch.Generator(device="cuda").manual_seed(7)
    values, scores = torch.randn((2, n, width), generator=g, device="cuda"), torch.randn((4, queries, k), generator=g, device="cuda")
    ids = torch.randint(1, n, (4, queries, k), generator=g, device="cuda")
    values[0, 0, 2] = value
    j = k - 1 if last else 0
    ids[0, 0, j], ids[1, 1, j] = 0, 0
    scores[0, 0, j], scores[1, 1, j] = -1e5, float("-inf")
    finite = certex.selected_attention(scores, ids, values, 1.0).isfinite()
    assert not finite[0, 0, 2] and finite.sum() == finite.numel() - 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [1.0, 100.0, 10_000.0])
@pytest.mark.parametrize("scale", [0.125, -0.125, 1.0, 0.0])
def test_attend_huge_scores(gpu, dtype, factor, scale):
    """Scores up to 4e10, far past where float32 has a fraction: alike, they weigh alike; next to the largest the others
    weigh nothing. A share and several, one wave's positions and all waves'."""
    lens, d, heads, kv, page = [3, 200, 9000], 64, 4, 2, 16
    kp, vp, table, _, values = paged(lens, page, kv, d, d, dtype, seed=31)
    kp[:] = -60_000.0
    q = torch.full((3, heads, d), factor, dtype=dtype, device="cuda")
    q[:, 1] = -factor
    out, lse = certex.paged_attention(q, kp, vp, table, torch.tensor(lens, device="cuda"), scale=scale, return_lse=True)
    low = float(torch.tensor(-60_000.0, dtype=dtype))
    for s, n in enumerate(lens):
        v = values[s].double().cpu()
        for h in range(heads):
            mean, spread = v[:, h // 2].mean(0), v[:, h // 2].abs().mean(0)
            score = scale * float(q[s, h, 0]) * low * d
            ref.assert_attended(out[s, h][None], mean[None], spread[None], torch.zeros(1), n, 1)
            want = score + math.log(n)
            assert abs(float(lse[s, h]) - want) <= 80 * U * (1 + abs(want))  # of 64 products and the logarithm's scale
    # one key less far down, or, where the sign is the other one's, all others
    kp[int(table[2, 70]), 5] = -40_000.0
    out = certex.paged_attention(q, kp, vp, table, torch.tensor(lens, device="cuda"), scale=scale)
    v = values[2].double().cpu()
    for h in range(heads):
        sign = scale * float(q[2, h, 0])
        if sign == 0:
            want, spread = v[:, h // 2].mean(0), v[:, h // 2].abs().mean(0)
        elif sign > 0:
            want = v[70 * page + 5, h // 2]
            spread = want.abs()
        else:
            rest = torch.cat([v[: 70 * page + 5, h // 2], v[70 * page + 6 :, h // 2]])
            want, spread = rest.mean(0), rest.abs().mean(0)
        ref.assert_attended(out[2, h][None], want[None], spread[None], torch.zeros(1), lens[2], 1)
