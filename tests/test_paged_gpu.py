"""The attention operators against their float64 definitions, with bounds from the number formats (paged_reference.py)."""

import math

import pytest
import torch

import libcertex_amd as certex
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ---- rotation ----


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d, r", [(128, 128), (80, 32), (64, 62), (34, 10), (256, 100), (7, 4), (2, 2), (24, 16)])
def test_rotate(gpu, dtype, layout, d, r):
    rope = certex.Rotary(d, rotary_dim=r, layout=layout, base=5000.0)
    x = rand(11, 5, d, dtype=dtype)
    p = ints([0, 1, 2, 3, 1000, 65_537, 131_071, 1_000_003, 7, 7, 8])
    y = rope(x, p)
    want = ref.rotate(x, p, rope.frequencies, layout, r)
    assert y.dtype == dtype and torch.equal(y[..., r:], x[..., r:])
    ref.assert_rotated(y, x, want, layout, r)
    back = rope(x, p, transpose=True)
    ref.assert_rotated(back, x, ref.rotate(x, p, rope.frequencies, layout, r, transpose=True), layout, r)


@pytest.mark.parametrize("tokens, heads", [(0, 3), (1, 1), (1, 64), (3000, 24)])
def test_rotate_sizes(gpu, tokens, heads):
    rope = certex.Rotary(96, scaling="ramp", factor=8.0, original_length=4096)
    x = rand(tokens, heads, 96, dtype=torch.bfloat16)
    p = torch.arange(tokens, device="cuda") * 37
    y = rope(x, p)
    assert y.shape == x.shape
    ref.assert_rotated(y, x, ref.rotate(x, p, rope.frequencies, "half", 96, rope.magnitude), "half", 96, rope.magnitude)


def test_rotate_any_position(gpu):
    """Angles are reduced exactly: positions past 2^32 and below 0 (float64 holds these products' fractions)."""
    rope = certex.Rotary(64)
    x = rand(6, 2, 64)
    p = ints([1 << 20, (1 << 31) + 5, (1 << 33) + 1, -1, -131_072, (1 << 24) + 1], torch.int64)
    # the reference's angles in extended precision: float64 loses 2^-20 of a turn at 2^33
    turns = [[float(((int(pos) * round(float(f) / (2 * math.pi) * 2**64)) % 2**64) / 2**64) for f in rope.frequencies]
             for pos in p.tolist()]
    angle = 2 * math.pi * torch.tensor(turns, dtype=torch.float64)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.double().cpu()[..., :32], x.double().cpu()[..., 32:]
    want = torch.cat([a * c - b * s, a * s + b * c], -1)
    ref.assert_rotated(rope(x, p), x, want, "half", 64)
    small = p.abs() < 1 << 21
    ref.assert_rotated(rope(x, p)[small], x[small], ref.rotate(x[small], p[small], rope.frequencies, "half", 64), "half", 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_strides(gpu, dtype, layout):
    rope = certex.Rotary(64, rotary_dim=48, layout=layout)
    p = torch.arange(9, device="cuda")
    keys = rand(4, 9, 64, dtype=dtype)  # head-major, as a KeyCache takes them
    want = ref.rotate(keys.transpose(0, 1), p, rope.frequencies, layout, 48)
    y = rope(keys.transpose(0, 1), p)
    ref.assert_rotated(y, keys.transpose(0, 1), want, layout, 48)
    wide = rand(9, 4, 200, dtype=dtype)
    for lo in (0, 1, 8):  # a slice of a fused projection: gaps between rows, any alignment
        x = wide[..., lo : lo + 64]
        ref.assert_rotated(rope(x, p), x, ref.rotate(x, p, rope.frequencies, layout, 48), layout, 48)
    gaps = wide[..., ::3][..., :64]  # gaps between elements
    ref.assert_rotated(rope(gaps, p), gaps, ref.rotate(gaps, p, rope.frequencies, layout, 48), layout, 48)
    one = rand(9, 1, 64, dtype=dtype).expand(9, 5, 64)
    ref.assert_rotated(rope(one, p), one, ref.rotate(one, p, rope.frequencies, layout, 48), layout, 48)
    batch = rand(3, 4, 7, 64, dtype=dtype).transpose(1, 2)  # (batch, tokens, heads, dim), heads first in memory
    bp = ints([[0, 1, 2, 3, 4, 5, 6], [9, 8, 7, 6, 5, 4, 3], [100, 200, 300, 400, 500, 600, 700]], torch.int64)
    ref.assert_rotated(rope(batch, bp), batch, ref.rotate(batch, bp, rope.frequencies, layout, 48), layout, 48)
    x = wide[..., :64].clone()
    before = x.clone()
    assert rope(x, p, out=x) is x  # in place
    ref.assert_rotated(x, before, ref.rotate(before, p, rope.frequencies, layout, 48), layout, 48)
    part = wide.clone()
    rope(part[..., 3:67], p, out=part[..., 100:164])
    ref.assert_rotated(part[..., 100:164], wide[..., 3:67], ref.rotate(wide[..., 3:67], p, rope.frequencies, layout, 48),
                       layout, 48)
    assert torch.equal(part[..., :100], wide[..., :100]) and torch.equal(part[..., 164:], wide[..., 164:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_gradient(gpu, layout):
    rope = certex.Rotary(40, rotary_dim=24, layout=layout, scaling="ramp", factor=4.0, original_length=512)
    p = torch.arange(50, device="cuda") * 11
    x, dy = rand(50, 3, 40).requires_grad_(), rand(50, 3, 40, seed=1)
    y = rope(x, p)
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    want = ref.rotate(dy, p, rope.frequencies, layout, 24, rope.magnitude, transpose=True)
    ref.assert_rotated(dx.detach(), dy, want, layout, 24, rope.magnitude)
    # differences: the rotation is linear, so any step gives the derivative up to rounding
    v = rand(50, 3, 40, seed=2)
    with torch.no_grad():
        slope = (((rope(x + v, p) - rope(x - v, p)).double() / 2) * dy).sum()
    size = float((v.double().abs() * dy.double().abs()).sum()) * rope.magnitude
    assert abs(float(slope - (dx.double() * v).sum())) <= 64 * 2.0**-24 * (size + float((x.detach().abs() * dy.abs()).sum()))
    # of a broadcast input, and of the gradient itself
    one = rand(50, 1, 40, seed=3).requires_grad_()
    (d1,) = torch.autograd.grad(rope(one.expand(50, 3, 40), p), one, dy)
    total = want.sum(1, keepdim=True)
    room = 32 * 2.0**-24 * rope.magnitude * 2 * dy.double().abs().cpu().amax(-1, keepdim=True).sum(1, keepdim=True)
    assert ((d1.double().cpu() - total).abs() <= room).all()
    dy2 = dy.clone().requires_grad_()
    (g,) = torch.autograd.grad(rope(x, p), x, dy2, create_graph=True)
    (gg,) = torch.autograd.grad(g, dy2, v)
    assert torch.equal(gg, rope(v, p))


# ---- paged cache ----


def paged(lens, page, kv, d, dv, dtype, seed=0, heads_first=False, spare=2, fill=float("nan"), capacity=None):
    """Pools whose unused slots hold `fill`, a shuffled table (-1 past a sequence), and every sequence's keys and
    values."""
    need = [-(-(n if capacity is None else max(n, capacity)) // page) for n in lens]
    pages = sum(need) + spare
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()

    def pool(width):
        if heads_first:
            return torch.full((pages, kv, page, width), fill, dtype=dtype, device="cuda").transpose(1, 2)
        return torch.full((pages, page, kv, width), fill, dtype=dtype, device="cuda")

    kp, vp = pool(d), pool(dv)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    keys, values, at = [], [], 0
    for s, n in enumerate(lens):
        table[s, : need[s]] = torch.tensor(order[at : at + need[s]], dtype=torch.int32)
        at += need[s]
        k, v = rand(n, kv, d, dtype=dtype, seed=seed + 10 * s), rand(n, kv, dv, dtype=dtype, seed=seed + 10 * s + 5)
        t = torch.arange(n)
        where = table[s].long()[t // page].cuda(), (t % page).cuda()
        kp[where], vp[where] = k, v
        keys.append(k)
        values.append(v)
    return kp, vp, table.cuda(), keys, values


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv, r, layout, page, heads_first", [
    (128, 128, 128, "half", 64, False), (64, 64, 64, "interleaved", 16, True), (80, 72, 32, "half", 24, False),
    (33, 17, 10, "interleaved", 5, True), (128, 128, 0, "half", 1, False),
])
def test_append(gpu, dtype, d, dv, r, layout, page, heads_first):
    old, new, kv, heads = [0, 7, 30, 64], [9, 1, 0, 20], 3, 6
    kp, vp, table, *_ = paged(old, page, kv, d, dv, dtype, heads_first=heads_first, fill=3.0, capacity=90)
    before_k, before_v = kp.clone(), vp.clone()
    seq = [s for s, n in enumerate(new) for _ in range(n)] + [1, -1, 99, 2]
    pos = [old[s] + i for s, n in enumerate(new) for i in range(n)] + [-1, 3, 3, 1 << 20]  # four that are not written
    t = len(pos)
    k, v, q = rand(t, kv, d, dtype=dtype), rand(t, kv, dv, dtype=dtype, seed=1), rand(t, heads, d, dtype=dtype, seed=2)
    rope = certex.Rotary(d, rotary_dim=r, layout=layout) if r else None
    out = certex.append_pages(k, v, kp, vp, table, ints(pos, torch.int64), sequences=ints(seq), rotary=rope, q=q)
    if rope is None:
        turned, q_want = k, q
        assert torch.equal(out, q)
    else:
        turned = rope(k, ints(pos))
        q_want = ref.rotate(q, ints(pos, torch.int64), rope.frequencies, layout, r)
        ref.assert_rotated(out, q, q_want, layout, r)
        ref.assert_rotated(turned, k, ref.rotate(k, ints(pos), rope.frequencies, layout, r), layout, r)
    host = table.cpu()
    for i in range(t - 4):
        at = int(host[seq[i], pos[i] // page]), pos[i] % page
        before_k[at], before_v[at] = turned[i], v[i]
    assert torch.equal(kp, before_k) and torch.equal(vp, before_v)


def test_append_strides_and_defaults(gpu):
    """Token t is sequence t; k, v and q are slices of one projection; a hole in the table; nothing without tokens."""
    kv, heads, d, page = 2, 4, 64, 16
    fused = rand(5, (heads + 2 * kv) * d, dtype=torch.bfloat16)
    q, k, v = (x.unflatten(1, (-1, d)) for x in fused.split([heads * d, kv * d, kv * d], 1))
    kp, vp, table, *_ = paged([0] * 5, page, kv, d, d, torch.bfloat16, fill=0.0, capacity=40)
    table[3, 1] = -1
    table[4, 0] = 10_000  # a page that the pool does not have
    pos = ints([0, 17, 39, 20, 3])
    rope = certex.Rotary(d)
    out = certex.append_pages(k, v, kp, vp, table, pos, rotary=rope, q=q)
    assert torch.equal(out, rope(q, pos))
    turned = rope(k, pos)
    for i, p in enumerate([0, 17, 39]):
        at = int(table[i, p // page]), p % page
        assert torch.equal(kp[at], turned[i]) and torch.equal(vp[at], v[i])
    assert int((kp != 0).any(-1).any(-1).sum()) == 3
    none = certex.append_pages(k[:0], v[:0], kp, vp, table, pos[:0], rotary=rope, q=q[:0])
    assert none.shape == (0, heads, d)


def check_attend(lens, heads, kv, d, dv, page, dtype, window=None, scale=None, loud=1.0, **kw):
    kp, vp, table, keys, values = paged(lens, page, kv, d, dv, dtype, **kw)
    q = rand(len(lens), heads, d, dtype=dtype, scale=loud)
    out, lse = certex.paged_attention(q, kp, vp, table, ints(lens), window=window, scale=scale, return_lse=True)
    assert out.shape == (len(lens), heads, dv) and out.dtype == dtype and lse.dtype == torch.float32
    for s, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        want, want_lse, spread, dots = ref.attend(q[s], keys[s][lo:], values[s][lo:], d**-0.5 if scale is None else scale)
        ref.assert_attended(out[s], want, spread, dots, n - lo, d, lse[s], want_lse)
    assert torch.equal(out, certex.paged_attention(q, kp, vp, table, ints(lens, torch.int64), window=window, scale=scale))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv", [(32, 8), (4, 4), (7, 1), (16, 1), (24, 1), (40, 2), (6, 2)])
def test_attend_heads(gpu, dtype, heads, kv):
    check_attend([1, 0, 33, 130, 700], heads, kv, 128, 128, 16, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", [(64, 64), (96, 96), (80, 72), (256, 256), (192, 128), (64, 256), (8, 8), (33, 17),
                                   (130, 66), (1, 1), (128, 40), (255, 255)])
def test_attend_dims(gpu, dtype, d, dv):
    check_attend([5, 64, 200, 31], 8, 4, d, dv, 32, dtype, seed=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 1000])
@pytest.mark.parametrize("heads_first", [False, True])
def test_attend_pages(gpu, dtype, page, heads_first):
    check_attend([1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 0, 500], 8, 2, 64, 64, page, dtype, heads_first=heads_first, seed=4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 5, 32, 100, 10_000])
def test_attend_window(gpu, dtype, window):
    check_attend([1, 0, 90, 101, 1000, 4000], 8, 2, 64, 64, 16, dtype, window=window, seed=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[20_000], [1, 9_000, 50], [3000] * 40, [0], [0, 0, 0]])
def test_attend_long(gpu, dtype, lens):
    check_attend(lens, 8, 2, 128, 128, 64, dtype, seed=6)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_extreme_scores(gpu, dtype):
    """Scores in the hundreds (one weight takes all), of a scale of 0 (all equal) and of a negative one."""
    check_attend([300, 5], 8, 2, 128, 128, 16, dtype, loud=30.0, seed=7)
    check_attend([300, 5], 8, 2, 128, 128, 16, dtype, scale=0.0, seed=8)
    check_attend([300, 5], 8, 2, 128, 128, 16, dtype, scale=-0.3, seed=9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fill", [float("inf"), float("-inf"), 0.0])
def test_attend_unused_slots(gpu, dtype, fill):
    """What slots past a length hold (NaN in the other tests) does not matter."""
    check_attend([1, 40, 63, 65], 8, 2, 64, 64, 32, dtype, fill=fill, seed=10)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_lowest_values(gpu, dtype):
    """Keys of the type's lowest value drive scores to -inf or far down: those positions weigh nothing, and a position
    of the largest finite score takes all."""
    lens = [70]
    kp, vp, table, keys, values = paged(lens, 16, 2, 64, 64, dtype, seed=11)
    q = torch.ones((1, 4, 64), dtype=dtype, device="cuda")
    low = torch.finfo(dtype).min
    for t in range(3, 70):
        at = int(table[0, t // 16]), t % 16
        kp[at] = low
    out, lse = certex.paged_attention(q, kp, vp, table, ints(lens), return_lse=True)
    want, want_lse, spread, dots = ref.attend(q[0], keys[0][:3], values[0][:3], 64**-0.5)
    ref.assert_attended(out[0], want, spread, dots, 70, 64, lse[0], want_lse)


def test_attend_lengths_and_holes(gpu):
    """Lengths below 0 and past the table are cut; positions of missing pages do not count."""
    dtype, page = torch.bfloat16, 16
    kp, vp, table, keys, values = paged([64, 64, 64, 64], page, 2, 64, 64, dtype, seed=12)
    q = rand(4, 4, 64, dtype=dtype)
    table[2, 1] = -1
    table[3, 0], table[3, 1], table[3, 2], table[3, 3] = -1, 10_000, -5, kp.shape[0]
    out, lse = certex.paged_attention(q, kp, vp, table, ints([-3, 1_000_000, 64, 64]), return_lse=True)
    assert (out[0] == 0).all() and (lse[0] == float("-inf")).all()
    assert (out[3] == 0).all() and (lse[3] == float("-inf")).all()
    want, want_lse, spread, dots = ref.attend(q[1], keys[1], values[1], 64**-0.5)
    ref.assert_attended(out[1], want, spread, dots, 64, 64, lse[1], want_lse)
    there = [t for t in range(64) if t // page != 1]
    want, want_lse, spread, dots = ref.attend(q[2], keys[2][there], values[2][there], 64**-0.5)
    ref.assert_attended(out[2], want, spread, dots, 48, 64, lse[2], want_lse)


def test_attend_nan_is_seen(gpu):
    """A NaN among the keys in use is not swallowed, and stays with its sequence and head."""
    kp, vp, table, *_ = paged([50, 50], 16, 2, 64, 64, torch.bfloat16, seed=13)
    kp[int(table[0, 1]), 3, 1, 5] = float("nan")
    out = certex.paged_attention(rand(2, 4, 64, dtype=torch.bfloat16), kp, vp, table, ints([50, 50]))
    assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and not out[1].isnan().any()

    q = rand(2, 4, 64, dtype=torch.bfloat16)
    q[1, 3] = float("nan")  # every score of a row
    for lens in ([50, 50], [50, 5000]):
        kp, vp, table, *_ = paged(lens, 16, 2, 64, 64, torch.bfloat16, seed=14)
        out, lse = certex.paged_attention(q, kp, vp, table, ints(lens), return_lse=True)
        assert out[1, 3].isnan().all() and lse[1, 3].isnan() and not out[0].isnan().any() and not out[1, :3].isnan().any()
    scores = torch.full((2, 1, 3000), float("nan"), device="cuda")
    scores[1] = 1.0
    out = certex.selected_attention(scores, torch.zeros((2, 1, 3000), dtype=torch.int64, device="cuda"), rand(2, 4, 64), 1.0)
    assert out[0].isnan().all() and not out[1].isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_value_is_seen(gpu, dtype):
    """An infinity among the values in use shows in its column, and in no other column, head or sequence."""
    kp, vp, table, *_ = paged([50, 50], 16, 2, 64, 64, dtype, seed=15)
    vp[int(table[0, 1]), 3, 1, 5] = float("inf")
    finite = certex.paged_attention(rand(2, 4, 64, dtype=dtype), kp, vp, table, ints([50, 50])).isfinite()
    assert not finite[0, 2:, 5].any() and finite.sum() == finite.numel() - 2

    # few queries a head gather rows; many, over values larger than a die's cache, go by ranges
    for queries, n, k in ((2, 500, 70), (64, 40_000, 2050)):
        values = rand(2, n, 64, dtype=dtype)
        values[1, 11, 5] = float("inf")
        ids = torch.randint(12, n, (4, queries, k), device="cuda")
        ids[2, 1, 9] = ids[3, 0, 0] = 11
        finite = certex.selected_attention(rand(4, queries, k), ids, values, 0.3).isfinite()
        assert not finite[2, 1, 5] and not finite[3, 0, 5] and finite.sum() == finite.numel() - 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_unaligned_queries(gpu, dtype):
    """Queries that are a slice of a projection (any alignment), pools with gaps between heads."""
    lens = [60, 200]
    kp, vp, table, keys, values = paged(lens, 16, 2, 64, 64, dtype, seed=14)
    wide = rand(2, 4, 200, dtype=dtype)
    both = torch.full((*kp.shape[:3], 131), float("nan"), dtype=dtype, device="cuda")
    both[..., 3:67], both[..., 67:] = kp, vp
    for q, k, v in [(wide[..., 1:65], kp, vp), (wide[..., 8:72], both[..., 3:67], both[..., 67:]),
                    (wide[..., ::3][..., :64], kp, both[..., 67:])]:
        out = certex.paged_attention(q, k, v, table, ints(lens))
        for s in range(2):
            want, _, spread, dots = ref.attend(q[s], keys[s], values[s], 64**-0.5)
            ref.assert_attended(out[s], want, spread, dots, lens[s], 64)


def test_offsets_past_32_bits(gpu):
    """Pages past 2^31 elements of a pool: appended to and attended over."""
    page, kv, d = 64, 8, 128
    pages = (1 << 31) // (page * kv * d) + 40
    kp = torch.empty((pages, page, kv, d), dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    table = ints([[pages - 1, 3, pages - 7], [0, pages - 2, pages - 30]])
    n = 150
    k, v = rand(2 * n, kv, d, dtype=torch.bfloat16), rand(2 * n, kv, d, dtype=torch.bfloat16, seed=1)
    pos, seq = torch.arange(n, device="cuda").repeat(2), torch.arange(2, device="cuda").repeat_interleave(n)
    certex.append_pages(k, v, kp, vp, table, pos, sequences=seq)
    assert torch.equal(kp[pages - 7, : n - 128], k[128:n]) and torch.equal(vp[pages - 30, : n - 128], v[n + 128 :])
    q = rand(2, 16, d, dtype=torch.bfloat16)
    out = certex.paged_attention(q, kp, vp, table, ints([n, n]))
    for s in range(2):
        want, _, spread, dots = ref.attend(q[s], k[s * n : (s + 1) * n], v[s * n : (s + 1) * n], d**-0.5)
        ref.assert_attended(out[s], want, spread, dots, n, d)
    scores = rand(16, 1, n)
    ids = torch.arange(n, device="cuda").expand(16, 1, n).contiguous()
    got = certex.selected_attention(scores, ids, vp, 0.7, page_table=table[0])
    for h in (0, 7, 15):
        w = torch.softmax(0.7 * scores[h, 0].double().cpu(), 0)
        rows = v[:n, h // 2].double().cpu()
        ref.assert_attended(got[h, 0][None], (w @ rows)[None], (w @ rows.abs())[None], 0.7 * scores[h, 0].abs().max()[None].cpu(), n, 1)


# ---- attention over a selected top k ----


def check_selected(scores, ids, rows_of, heads, kv, scale, out, lse):
    """rows_of(g): values of head g in float64, (n, dv)."""
    for h in range(heads):
        values = rows_of(h // (heads // kv))
        for i in range(scores.shape[1]):
            j, s = ids[h, i].cpu().long(), scale * scores[h, i].double().cpu()
            keep = (j >= 0) & (j < values.shape[0]) & (scores[h, i].cpu() > float("-inf"))
            j, s = j[keep], s[keep]
            if len(j) == 0:
                assert (out[h, i] == 0).all() and lse[h, i] == float("-inf")
                continue
            w, rows = torch.softmax(s, 0), values[j]
            ref.assert_attended(out[h, i][None], (w @ rows)[None], (w @ rows.abs())[None], s.abs().max()[None], len(j), 1,
                                lse[h, i][None], torch.logsumexp(s, 0)[None])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 3, 64, 257, 2048, 5000])
@pytest.mark.parametrize("dv, heads, kv, m", [(128, 4, 2, 3), (72, 3, 1, 2), (17, 2, 2, 1), (256, 4, 4, 1)])
def test_selected(gpu, dtype, k, dv, heads, kv, m):
    n = 6000
    values = rand(kv, n, dv, dtype=dtype)
    scores = rand(heads, m, k, scale=11.0).sort(-1, descending=True).values
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.rand((heads, m, n), generator=g, device="cuda").topk(k, -1).indices
    out, lse = certex.selected_attention(scores, ids, values, 0.09, return_lse=True)
    assert out.shape == (heads, m, dv) and out.dtype == dtype
    host = values.double().cpu()
    check_selected(scores, ids, lambda j: host[j], heads, kv, 0.09, out, lse)
    narrow = certex.selected_attention(scores[:, 0], ids[:, 0].to(torch.int32), values, 0.09)
    assert torch.equal(narrow, out[:, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [512, 700, 2048, 2100, 4097])
@pytest.mark.parametrize("dv", [128, 62, 200])
def test_selected_shared_rows(gpu, dtype, k, dv):
    """Queries of a head that select more rows than it has, of more than a die's cache; ids repeated within a query; all in
    one range."""
    n, heads, kv, m = 35_000, 4, 2, 64
    values = rand(kv, n, dv, dtype=dtype)
    scores = rand(heads, m, k, scale=5.0)
    ids = torch.randint(0, n, (heads, m, k), device="cuda")
    ids[0, 1] = 17
    ids[0, 2] = ids[0, 2] % 500
    ids[1, 0] = -1
    ids[1, 1, ::2] = n
    ids[1, 2, 1:] = -1
    ids[2, 3, : k // 2] = -5
    scores[3, 4] = scores[3, 4].sort(descending=True).values * 100
    out, lse = certex.selected_attention(scores, ids, values, 0.3, return_lse=True)
    host = values.double().cpu()
    few = [0, 1, 2, 3, 4, m - 1]
    check_selected(scores[:, few], ids[:, few], lambda j: host[j], heads, kv, 0.3, out[:, few], lse[:, few])
    assert torch.equal(out, certex.selected_attention(scores, ids, values, 0.3))


@pytest.mark.parametrize("dtype", TYPES)
def test_selected_missing(gpu, dtype):
    """-1 and ids past the values, scores of -inf, rows of none; values that nobody selected hold NaN."""
    values = rand(2, 500, 64, dtype=dtype)
    values[:, 250:] = float("nan")
    scores, ids = rand(4, 5, 96), torch.randint(0, 250, (4, 5, 96), device="cuda")
    ids[:, 1, ::3] = -1
    ids[:, 2, 5:] = -1
    ids[:, 3] = -1
    ids[0, 4, :7], scores[1, 4, 9:20], scores[2, 4] = 500, float("-inf"), float("-inf")
    scores[1, 1, ::3] = float("-inf")
    ids[1, 4, 9:20] = 400  # a NaN row of weight 0
    scores[3, 1, ::3] = float("nan")  # of missing ids
    out, lse = certex.selected_attention(scores, ids, values, 1.0, return_lse=True)
    host = values.double().cpu()
    check_selected(scores, ids, lambda j: host[j], 4, 2, 1.0, out, lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_selected_paged(gpu, dtype, page):
    n, kv = 300, 2
    _, vp, table, _, values = paged([n], page, kv, 8, 80, dtype, heads_first=True, seed=15)
    scores = rand(4, 6, 100)
    ids = torch.rand((4, 6, n), device="cuda").topk(100, -1).indices
    table = table[0].contiguous()
    gone = table.clone()
    gone[0] = -1
    out, lse = certex.selected_attention(scores, ids, vp, 0.5, page_table=table, return_lse=True)
    host = values[0].double().cpu()
    check_selected(scores, ids, lambda g: host[:, g], 4, kv, 0.5, out, lse)
    out, lse = certex.selected_attention(scores, ids, vp, 0.5, page_table=gone, return_lse=True)
    check_selected(scores, torch.where(ids < page, -1, ids), lambda g: host[:, g], 4, kv, 0.5, out, lse)


def test_selected_strides_and_empty(gpu):
    values = rand(500, 2, 200, dtype=torch.float16).transpose(0, 1)[..., 5:69]
    scores, ids = rand(4, 3, 40), torch.randint(0, 500, (4, 3, 40), device="cuda")
    out, lse = certex.selected_attention(scores, ids, values, -0.4, return_lse=True)
    host = values.double().cpu()
    check_selected(scores, ids, lambda j: host[j], 4, 2, -0.4, out, lse)
    out, lse = certex.selected_attention(scores[..., :0], ids[..., :0], values, 1.0, return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()
    assert certex.selected_attention(scores[:, :0], ids[:, :0], values, 1.0).shape == (4, 0, 64)


def test_key_cache_attend(gpu):
    """Attention over the exact top k of a KeyCache; with k the whole cache it is dense attention over the pages."""
    kv, heads, n, d, m = 2, 8, 700, 64, 3
    kp, vp, table, keys, values = paged([n], 16, kv, d, d, torch.bfloat16, seed=16)
    q = rand(heads, m, d, dtype=torch.bfloat16)
    cache = certex.KeyCache(kv, d, k=100).append(keys[0].transpose(0, 1))
    got = cache.attend(q, values[0].transpose(0, 1))
    scores, ids = cache.topk(q)
    assert torch.equal(got, certex.selected_attention(scores, ids, values[0].transpose(0, 1), d**-0.5))
    assert torch.equal(got, cache.attend(q, vp, page_table=table[0]))
    whole = cache.attend(q, vp, k=n, page_table=table[0])
    for i in range(m):
        dense = certex.paged_attention(q[:, i][None], kp, vp, table, ints([n]))
        for x in (whole[:, i], dense[0]):
            want, _, spread, dots = ref.attend(q[:, i], keys[0], values[0], d**-0.5)
            ref.assert_attended(x, want, spread, dots, n, d)
    assert torch.equal(cache.attend(q[:, 0], vp, page_table=table[0]), got[:, 0])


# ---- streams, graphs, refusals ----


def test_other_streams(gpu):
    """Calls follow torch's current stream, whatever stream ran before."""
    lens = [5000, 300]
    kp, vp, table, keys, values = paged(lens, 16, 2, 64, 64, torch.bfloat16, seed=17)
    q = rand(2, 8, 64, dtype=torch.bfloat16)
    want = certex.paged_attention(q, kp, vp, table, ints(lens))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            late = torch.zeros_like(q)
            for _ in range(20):
                late += 0.0 * rand(2, 8, 64)
            late += q  # the queries are ready only at the end of this stream's work
            outs.append(certex.paged_attention(late, kp, vp, table, ints(lens)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_graph(gpu):
    """One decoding step recorded as a graph: append with rotation, dense and sparse attention; replayed with other
    inputs, eager work in between."""
    kv, heads, d, page = 2, 8, 64, 16
    kp, vp, table, *_ = paged([0, 0], page, kv, d, d, torch.bfloat16, fill=0.0, capacity=2000)
    rope = certex.Rotary(d)
    pos = ints([0, 0])
    q, k, v = (rand(2, h, d, dtype=torch.bfloat16) for h in (heads, kv, kv))
    scores, ids = rand(heads, 1, 50), torch.randint(0, 30, (heads, 1, 50), device="cuda")

    def step():
        turned = certex.append_pages(k, v, kp, vp, table, pos, rotary=rope, q=q)
        dense = certex.paged_attention(turned, kp, vp, table, pos + 1)
        return dense, certex.selected_attention(scores, ids, vp, 0.125, page_table=table[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, p in enumerate([0, 1, 37, 38, 1500]):
        pos.copy_(ints([p, p // 2]))
        for x, h, s in ((q, heads, 1), (k, kv, 2), (v, kv, 3)):
            x.copy_(rand(2, h, d, dtype=torch.bfloat16, seed=100 * i + s))
        graph.replay()
        got = [x.clone() for x in out]
        pools = kp.clone(), vp.clone()
        torch.cuda.synchronize()
        want = step()  # writes the same keys and values again
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(kp, pools[0]) and torch.equal(vp, pools[1])
        rand(1000, 1000).sum().item()


def test_refusals(gpu):
    rope = certex.Rotary(64)
    x, p = rand(5, 2, 64), ints([0, 1, 2, 3, 4])
    pool, table = torch.zeros(3, 8, 2, 64, device="cuda"), torch.zeros(5, 3, dtype=torch.int32, device="cuda")
    scores, ids, values = rand(2, 1, 4), torch.zeros(2, 1, 4, dtype=torch.int64, device="cuda"), rand(2, 9, 64)
    grad = x.clone().requires_grad_()
    for call, match in [
        (lambda: rope(x[..., :32], p), "x must be"), (lambda: rope(x, p[:4]), "one entry per token"),
        (lambda: rope(x, p.float()), "int32 or torch.int64"), (lambda: rope(x.double(), p), "float32, float16 or bfloat16"),
        (lambda: rope(x, p, out=x.half()), "out must be"), (lambda: rope(x, p, out=x[:4]), "shape of x"),
        (lambda: rope(x, p, out=x[:, :1].expand(5, 2, 64)), "broadcast"), (lambda: rope(grad, p, out=x), "no out"),
        (lambda: certex.append_pages(x, x, pool, pool.half(), table, p), "v_pages must be"),
        (lambda: certex.append_pages(x, x[:4], pool, pool, table, p), "tokens and heads"),
        (lambda: certex.append_pages(x, x, pool[:, :, :1], pool, table, p), "k_pages must have shape"),
        (lambda: certex.append_pages(x, x, pool, pool, table[:4], p), "one row per token"),
        (lambda: certex.append_pages(x, x, pool, pool, table, p, rotary=certex.Rotary(32)), "heads of 32"),
        (lambda: certex.append_pages(x, x, pool, pool, table, p, q=x[:4]), "q must have the tokens"),
        (lambda: certex.append_pages(grad, x, pool, pool, table, p), "no gradient"),
        (lambda: certex.append_pages(x, x, pool[:1].expand(3, 8, 2, 64), pool, table, p), "broadcast"),
        (lambda: certex.append_pages(x, x, pool, pool, table.long(), p), "int32"),
        (lambda: certex.paged_attention(x, pool, pool, table, p, window=0), "window"),
        (lambda: certex.paged_attention(x, pool, pool, table, p[:3]), "lengths must have shape"),
        (lambda: certex.paged_attention(x, pool, pool, table, p, scale=float("nan")), "finite"),
        (lambda: certex.paged_attention(grad, pool, pool, table, p), "no gradient"),
        (lambda: certex.paged_attention(x.half(), pool, pool, table, p), "float16"),
        (lambda: certex.selected_attention(scores.half(), ids, values, 1.0), "float32 GPU tensor"),
        (lambda: certex.selected_attention(scores, ids[..., :3], values, 1.0), "one shape"),
        (lambda: certex.selected_attention(scores, ids, values[0], 1.0), "3 dimensions"),
        (lambda: certex.selected_attention(scores, ids, pool, 1.0, page_table=table), "one sequence's pages"),
        (lambda: certex.selected_attention(scores, ids, values.requires_grad_(), 1.0), "no gradient"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d, r", [(130, 66), (128, 102), (61, 34), (45, 44), (20, 18), (17, 16), (9, 8)])
def test_rotate_moved_vectors(gpu, dtype, layout, d, r):
    """Rows that are no whole vectors, aligned and not, written elsewhere and in place."""
    rope = certex.Rotary(d, rotary_dim=r, layout=layout)
    p = torch.arange(40, device="cuda") * 977
    wide = rand(40, 3, d + 9, dtype=dtype)
    for lo in (0, 3):
        x = wide[..., lo : lo + d]
        want = ref.rotate(x, p, rope.frequencies, layout, r)
        y = rope(x, p)
        ref.assert_rotated(y, x, want, layout, r)
        held = wide.clone()
        part = held[..., lo : lo + d]
        assert rope(part, p, out=part) is part and torch.equal(part, y)
        assert torch.equal(held[..., :lo], wide[..., :lo]) and torch.equal(held[..., lo + d :], wide[..., lo + d :])
    kp = torch.zeros((6, 8, 3, d), dtype=dtype, device="cuda")
    vp = torch.zeros((6, 8, 3, d + 9), dtype=dtype, device="cuda")
    table = ints([[4, 0, 5, 1, 3]])
    x, at = wide[..., 3 : 3 + d], torch.arange(40, device="cuda")
    certex.append_pages(x, wide, kp, vp, table, at, sequences=torch.zeros_like(at), rotary=rope)
    page, slot = table[0].long()[at // 8], at % 8
    assert torch.equal(kp[page, slot], rope(x, at)) and torch.equal(vp[page, slot], wide)


def test_gradient_outlives_its_rotation(gpu):
    """A graph keeps the frequencies that its backward needs."""
    x, p = rand(9, 2, 32).requires_grad_(), torch.arange(9, device="cuda") * 5
    rope = certex.Rotary(32)
    f = rope.frequencies
    y = rope(x, p)
    del rope
    dy = rand(9, 2, 32, seed=1)
    y.backward(dy)
    ref.assert_rotated(x.grad, dy, ref.rotate(dy, p, f, "half", 32, transpose=True), "half", 32)


def test_threads(gpu):
    """Calls of several threads at once, each on a stream of its own; the rotation and its frequencies are shared."""
    import threading

    lens = [900, 40]
    kp, vp, table, *_ = paged(lens, 16, 2, 64, 64, torch.bfloat16, seed=18)
    rope, pos = certex.Rotary(64), ints([899, 39])
    qs = [rand(2, 8, 64, dtype=torch.bfloat16, seed=100 + i) for i in range(4)]
    want = [certex.paged_attention(rope(q, pos), kp, vp, table, ints(lens)) for q in qs]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(50):
                    got = certex.paged_attention(rope(qs[i], pos), kp, vp, table, ints(lens))
                    if not torch.equal(got, want[i]):
                        failed.append(i)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
