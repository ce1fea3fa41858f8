"""4-bit pages against their definition (packed_reference.py): what they hold, and the attention over them."""

import pytest
import torch

import libcertex_amd as certex
from tests import packed_reference as pack
from tests import shaped_reference as ref
from tests.test_paged_gpu import ints, rand
from tests.test_prompt_gpu import slopes_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
DIMS = [(128, 128), (64, 64), (96, 96), (192, 192), (256, 256), (80, 72), (192, 128), (64, 256), (256, 40), (33, 17), (130, 66),
        (1, 1), (255, 200), (97, 160), (8, 129)]


def weight_unit(dtype):
    """Weights times scales meet the codes rounded to float16, or as two such elements for float32, the second cut; their product is
    rounded once before."""
    return (2.0**-21 if dtype == torch.float32 else 2.0**-11) + 2.0**-24


def packed(lens, page, kv, d, dv, dtype, seed=0, spare=2, fill=0xff, capacity=None):
    """Pages whose unused bytes are `fill` (scales and offsets of NaN), a shuffled table, and every sequence's keys and values."""
    need = [-(-(n if capacity is None else max(n, capacity)) // page) for n in lens]
    pages = certex.PackedPages(sum(need) + spare, page, kv, d, dv)
    pages.data.fill_(fill)
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    table = table.cuda()
    t = sum(lens)
    k, v = rand(t, kv, d, dtype=dtype, seed=seed), rand(t, kv, dv, dtype=dtype, seed=seed + 1)
    k[..., :: max(1, d // 4)] *= 4
    positions = torch.cat([torch.arange(n) for n in lens]).cuda()
    sequences = torch.arange(len(lens)).repeat_interleave(torch.tensor(lens)).cuda()
    pages.append(k, v, table, positions, sequences=sequences)
    return pages, table, k, v, positions, sequences


def check_read(pages, table, positions, sequences, k, v, dtype):
    """The pages hold what the definition says: exactly, rounded once to float32 and once more to a 16-bit type."""
    got_k, got_v = pages.read(table, positions, sequences=sequences, dtype=dtype)
    for got, x in ((got_k, k), (got_v, v)):
        want = pack.stored(x)[0].float().to(dtype)
        assert got.dtype == dtype and torch.equal(got.cpu().nan_to_num(7.5), want.nan_to_num(7.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", DIMS)
def test_held(gpu, dtype, d, dv):
    pages, table, k, v, positions, sequences = packed([1, 0, 33, 70], 16, 3, d, dv, dtype)
    check_read(pages, table, positions, sequences, k, v, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [8, 24, 64, 1000])
def test_held_pages(gpu, dtype, page):
    pages, table, k, v, positions, sequences = packed([5, 64, 200], page, 2, 64, 80, dtype, seed=1)
    check_read(pages, table, positions, sequences, k, v, dtype)
    for other in TYPES:
        check_read(pages, table, positions.int(), sequences.int(), k, v, other)


@pytest.mark.parametrize("dtype", TYPES)
def test_held_extremes(gpu, dtype):
    """Constant groups, zeros, both zeros' signs, subnormal and tiny spreads, the type's largest, infinities and NaN; halves
    between codes go to the even one."""
    d = 128
    big = torch.finfo(dtype).max
    rows = [torch.zeros(d), torch.full((d,), -3.25), torch.full((d,), 1.0e-7), torch.linspace(0, 1e-6, d), torch.linspace(-1e-4, 1e-4, d),
            torch.linspace(-big, big, d), torch.full((d,), big), torch.linspace(-60000, 60000, d), torch.linspace(0, 9e5, d)]
    halves = torch.arange(d) % 31 * 0.5  # 0, 0.5, ..., 15: scale 1
    rows += [halves, -halves, halves * 0.25 + 2]
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = torch.linspace(-1, 1, d)
        x[70] = bad
        rows.append(x)
    k = torch.stack(rows)[:, None].to(dtype).cuda()
    pages = certex.PackedPages(4, 8, 1, d)
    table, positions = ints([[2, 0, 3, 1]]), torch.arange(k.shape[0], device="cuda")
    sequences = torch.zeros_like(positions)
    pages.append(k, -k, table, positions, sequences=sequences)
    check_read(pages, table, positions, sequences, k, -k, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, r, layout", [(128, 128, "half"), (64, 48, "interleaved"), (80, 32, "half"), (33, 10, "interleaved"),
                                          (256, 250, "half")])
def test_append_turned(gpu, dtype, d, r, layout):
    """Keys that are turned on the way are those that the rotation gives, bit for bit."""
    rope = certex.Rotary(d, rotary_dim=r, layout=layout, scaling="ramp", factor=4.0, original_length=64)
    k, v = rand(40, 3, d, dtype=dtype), rand(40, 3, d, dtype=dtype, seed=1)
    table, positions = ints([[3, 1, 0], [2, 5, 4]]), torch.arange(40, device="cuda") % 20
    sequences = torch.arange(40, device="cuda") // 20
    one, two = certex.PackedPages(6, 8, 3, d), certex.PackedPages(6, 8, 3, d)
    one.append(k, v, table, positions, sequences=sequences, rotary=rope)
    two.append(rope(k, positions), v, table, positions, sequences=sequences)
    assert torch.equal(one.data, two.data) and one.data.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_append_skips_and_strides(gpu, dtype):
    """Padding, missing pages and other slots stay as they are; slices of a projection; token t is sequence t."""
    kv, d = 2, 64
    fused = rand(6, 4 * kv * d, dtype=dtype)
    k, v = (x.unflatten(1, (-1, d)) for x in (fused[:, 5 : 5 + kv * d], fused[:, 3 * kv * d :]))
    pages = certex.PackedPages(8, 16, kv, d)
    pages.data.copy_(torch.arange(pages.data.numel(), device="cuda").view_as(pages.data) % 251)
    before = pages.data.clone()
    table = ints([[0, 1], [2, -1], [3, 4], [5, 6], [100, 7], [-7, 7]])
    positions = ints([17, 20, -1, 32, 3, 5])  # of these the first alone has a slot
    pages.append(k, v, table, positions)
    got = pages.read(table, positions)
    assert (got[0][1:] == 0).all() and (got[1][1:] == 0).all()
    changed = (pages.data != before).any(-1).nonzero().tolist()
    assert changed == [[1, 0, 0], [1, 1, 0]]
    check_read(pages, table[:1], positions[:1], None, k[:1], v[:1], dtype)
    # within the records only that slot: the others' elements are as before
    others = ints([16, 18, 19, 20, 21, 22, 23])
    zeros = torch.zeros_like(others)
    after = pages.read(table, others, sequences=zeros, dtype=torch.float32)
    pages.data.copy_(before)
    for x, y in zip(after, pages.read(table, others, sequences=zeros, dtype=torch.float32)):
        assert torch.equal(x.nan_to_num(7.5), y.nan_to_num(7.5))
    pages.append(k[:0], v[:0], table, positions[:0])
    assert pages.read(table, positions[:0])[0].shape == (0, kv, d) and torch.equal(pages.data, before)


def check_attend(lens, heads, kv, d, dv, page, dtype, seed=0, loud=1.0, scale=None, **how):
    pages, table, k, v, positions, sequences = packed(lens, page, kv, d, dv, dtype, seed=seed)
    q = rand(len(lens), heads, d, dtype=dtype, scale=loud, seed=seed + 2)
    out, lse = pages.attend(q, table, ints(lens), return_lse=True, scale=scale, **how)
    assert out.shape == (len(lens), heads, dv) and out.dtype == dtype and lse.dtype == torch.float32
    at = 0
    for s, n in enumerate(lens):
        (keys, key_sizes), (values, value_sizes) = (pack.stored(x[at : at + n]) for x in (k, v))
        at += n
        want = ref.attend(q[s : s + 1], torch.tensor([n - 1]), keys, values, d**-0.5 if scale is None else scale, weight=weight_unit(dtype),
                          key_sizes=key_sizes, value_sizes=value_sizes, **how)
        ref.check(out[s : s + 1], lse[s : s + 1], want)
    assert torch.equal(out, pages.attend(q, table, ints(lens, torch.int64), scale=scale, **how))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv", [(32, 8), (4, 4), (7, 1), (16, 1), (24, 1), (40, 2), (6, 2)])
def test_attend_heads(gpu, dtype, heads, kv):
    check_attend([1, 0, 33, 130, 700], heads, kv, 128, 128, 16, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", DIMS)
def test_attend_dims(gpu, dtype, d, dv):
    check_attend([5, 64, 200, 31], 8, 4, d, dv, 32, dtype, seed=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 1000])
def test_attend_pages(gpu, dtype, page):
    check_attend([1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 0, 500], 8, 2, 64, 64, page, dtype, seed=4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 5, 32, 100, 10_000])
def test_attend_window(gpu, dtype, window):
    check_attend([1, 0, 90, 101, 1000, 4000], 8, 2, 64, 64, 16, dtype, window=window, seed=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap, lean, window", [(5.0, False, None), (50.0, True, 90), (None, True, None)])
def test_attend_bent(gpu, dtype, cap, lean, window):
    check_attend([1, 0, 33, 130, 700], 8, 2, 128, 128, 16, dtype, cap=cap, slopes=slopes_of(8) if lean else None, window=window,
                 loud=4.0, seed=6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[20_000], [1, 9_000, 50], [3000] * 40, [0], [0, 0, 0]])
def test_attend_long(gpu, dtype, lens):
    check_attend(lens, 8, 2, 128, 128, 64, dtype, seed=7)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_extreme_scores(gpu, dtype):
    """Scores in the hundreds (one weight takes all), of a scale of 0 (all equal) and of a negative one."""
    check_attend([300, 5], 8, 2, 128, 128, 16, dtype, loud=30.0, seed=8)
    check_attend([300, 5], 8, 2, 128, 128, 16, dtype, scale=0.0, seed=9)
    check_attend([300, 5], 8, 2, 128, 128, 16, dtype, scale=-0.3, seed=10)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e4])
def test_attend_value_sizes(gpu, dtype, size):
    """Values of any size, and that grow and shrink along a sequence; queries of any size. float16 scales hold steps down to 6e-8."""
    n, kv, d = 700, 2, 128
    pages = certex.PackedPages(44, 16, kv, d)
    table = torch.randperm(44, generator=torch.Generator().manual_seed(1)).int()[None].cuda()
    k, v = rand(n, kv, d, dtype=dtype), rand(n, kv, d, dtype=dtype, seed=1)
    v *= size
    v[::7] *= 0.01
    v[300:400] *= 3
    v[500] = 0
    v[:, 0] *= torch.logspace(-2, 0, n, device="cuda").to(dtype)[:, None]
    positions = torch.arange(n, device="cuda")
    pages.append(k, v, table, positions, sequences=torch.zeros_like(positions))
    (keys, key_sizes), (values, value_sizes) = pack.stored(k), pack.stored(v)
    for loud in (1.0, 1e-20, 1e20) if dtype == torch.float32 else (1.0,):
        q = rand(1, 8, d, dtype=dtype, seed=2, scale=loud)
        scale = d**-0.5 / loud
        out, lse = pages.attend(q, table, ints([n]), scale=scale, return_lse=True)
        ref.check(out, lse, ref.attend(q, torch.tensor([n - 1]), keys, values, scale, weight=weight_unit(dtype), key_sizes=key_sizes,
                                       value_sizes=value_sizes))


@pytest.mark.parametrize("fill", [0x00, 0x7f, 0x7c])
def test_attend_unused_bytes(gpu, fill):
    """What unused slots hold (scales of NaN in the other tests; infinite ones here) does not matter."""
    pages, table, *_ = packed([1, 40, 63, 65], 32, 2, 64, 64, torch.bfloat16, fill=0xff, seed=11)
    other, same, *_ = packed([1, 40, 63, 65], 32, 2, 64, 64, torch.bfloat16, fill=fill, seed=11)
    q = rand(4, 4, 64, dtype=torch.bfloat16)
    out = [p.attend(q, table, ints([1, 40, 63, 65])) for p in (pages, other)]
    assert torch.equal(*out) and out[0].isfinite().all()


def test_attend_lengths_and_holes(gpu):
    """Lengths below 0 and past the table are cut; positions of missing pages do not count."""
    dtype, page = torch.bfloat16, 16
    pages, table, k, v, *_ = packed([64] * 4, page, 2, 64, 64, dtype, seed=12)
    q = rand(4, 4, 64, dtype=dtype)
    table[2, 1] = -1
    table[3] = ints([-1, 10_000, -5, pages.data.shape[0]])
    out, lse = pages.attend(q, table, ints([-3, 1_000_000, 64, 64]), return_lse=True)
    assert (out[[0, 3]] == 0).all() and (lse[[0, 3]] == float("-inf")).all()
    for s, there in ((1, None), (2, torch.arange(64) // page != 1)):
        (keys, key_sizes), (values, value_sizes) = (pack.stored(x[64 * s : 64 * s + 64]) for x in (k, v))
        ref.check(out[s : s + 1], lse[s : s + 1],
                  ref.attend(q[s : s + 1], torch.tensor([63]), keys, values, 64**-0.5, weight=weight_unit(dtype), key_sizes=key_sizes,
                             value_sizes=value_sizes, there=there))


def test_attend_nan_is_seen(gpu):
    """NaN among keys, values or queries shows where it counts, and in no other sequence or head (of a value: in its 64
    columns)."""
    n, kv, d = 50, 2, 128
    table = ints([[0, 1, 2, 3], [4, 5, 6, 7]])
    positions, sequences = torch.arange(2 * n, device="cuda") % n, torch.arange(2 * n, device="cuda") // n
    k, v = rand(2 * n, kv, d, dtype=torch.bfloat16), rand(2 * n, kv, d, dtype=torch.bfloat16, seed=1)
    q = rand(2, 4, d, dtype=torch.bfloat16)
    for x in (k, v):
        keep = x[20, 1, 70].clone()
        x[20, 1, 70] = float("nan")
        pages = certex.PackedPages(8, 16, kv, d)
        pages.append(k, v, table, positions, sequences=sequences)
        x[20, 1, 70] = keep
        out = pages.attend(q, table, ints([n, n]))
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[0, 2:, 0 if x is k else 64 :] = True
        assert out[bad].isnan().all() and out[~bad].isfinite().all()
    pages = certex.PackedPages(8, 16, kv, d)
    pages.append(k, v, table, positions, sequences=sequences)
    q[1, 3, 5] = float("nan")
    out, lse = pages.attend(q, table, ints([n, n]), return_lse=True)
    assert out[1, 3].isnan().all() and lse[1, 3].isnan() and int(out.isnan().sum()) == d


def test_offsets_past_32_bits(gpu):
    """Pages past 2^32 bytes of a pool: appended to, read and attended over."""
    page, kv, d = 64, 8, 128
    n_pages = (1 << 32) // (page // 8 * kv * 1152) + 40
    data = torch.empty((n_pages, kv, page // 8, 1152), dtype=torch.uint8, device="cuda")
    pages = certex.PackedPages(n_pages, page, kv, d, data=data)
    table, n = ints([[n_pages - 1, 3, n_pages - 7], [0, n_pages - 2, n_pages - 30]]), 150
    k, v = rand(2 * n, kv, d, dtype=torch.bfloat16), rand(2 * n, kv, d, dtype=torch.bfloat16, seed=1)
    positions, sequences = torch.arange(n, device="cuda").repeat(2), torch.arange(2, device="cuda").repeat_interleave(n)
    pages.append(k, v, table, positions, sequences=sequences)
    check_read(pages, table, positions, sequences, k, v, torch.bfloat16)
    q = rand(2, 16, d, dtype=torch.bfloat16)
    out = pages.attend(q, table, ints([n, n]))
    for s in range(2):
        (keys, key_sizes), (values, value_sizes) = (pack.stored(x[s * n : s * n + n]) for x in (k, v))
        ref.check(out[s : s + 1], None, ref.attend(q[s : s + 1], torch.tensor([n - 1]), keys, values, d**-0.5, weight=weight_unit(torch.bfloat16),
                                                  key_sizes=key_sizes, value_sizes=value_sizes))


def test_refusals(gpu):
    pages, table, k, v, positions, sequences = packed([20, 20], 16, 2, 64, 48, torch.bfloat16, seed=13)
    q, lens = rand(2, 4, 64, dtype=torch.bfloat16), ints([20, 20])

    def append(k=k, v=v, table=table, positions=positions, sequences=sequences, **kw):
        pages.append(k, v, table, positions, sequences=sequences, **kw)

    def attend(q=q, table=table, lens=lens, **kw):
        return pages.attend(q, table, lens, **kw)

    append(), attend(), pages.read(table, positions, sequences=sequences)
    for call, kw, match in [
        (append, dict(k=k[:, :1]), "heads of the pages"), (append, dict(v=v[:5]), "tokens and heads of k"),
        (append, dict(k=k[..., :32]), "of heads of 64"), (append, dict(v=k), "values of 48"), (append, dict(v=v.float()), "as the other"),
        (append, dict(positions=positions[:3]), "positions must have shape"), (append, dict(sequences=None), "one row per token"),
        (append, dict(sequences=sequences[:3]), "sequences must have shape"), (append, dict(k=k.cpu()), "GPU"),
        (append, dict(k=k.clone().requires_grad_()), "no gradient"), (append, dict(rotary=certex.Rotary(128)), "of heads of 128"),
        (append, dict(table=table.long()), "int32"), (append, dict(k=k.double()), "float32, float16 or bfloat16"),
        (attend, dict(q=q[:, :3]), "multiple of the key heads"), (attend, dict(q=q[..., :32]), "of heads of 64"),
        (attend, dict(q=q[:1]), "one row per sequence"), (attend, dict(lens=lens[:1]), "lengths must have shape"),
        (attend, dict(q=q.clone().requires_grad_()), "no gradient"), (attend, dict(window=0), "at least 1"),
        (attend, dict(cap=-2.0), "positive"), (attend, dict(slopes=slopes_of(3)), "slopes must have shape"),
        (attend, dict(scale=float("nan")), "finite"), (attend, dict(q=q.double()), "float32, float16 or bfloat16"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
    for kw, match in [(dict(positions=positions[None]), "1 dimension"), (dict(dtype=torch.int32), "float32, float16 or bfloat16"),
                      (dict(dtype="bfloat16"), "torch.dtype"), (dict(sequences=sequences[:2]), "sequences must have shape")]:
        with pytest.raises(ValueError, match=match):
            pages.read(**{**dict(page_table=table, positions=positions, sequences=sequences), **kw})
    for args, kw in [((4, 12, 2, 64), {}), ((4, 0, 2, 64), {}), ((-1, 8, 2, 64), {}), ((4, 8, 0, 64), {}), ((4, 8, 2, 257), {}),
                     ((4, 8, 2, 0), {}), ((4, 8, 2, 64, 300), {}), ((4, 8, 2, 64), dict(data=pages.data)),
                     ((4, 8, 2, 64), dict(data=torch.zeros(4, 2, 1, 576, dtype=torch.uint8)))]:
        with pytest.raises(ValueError):
            certex.PackedPages(*args, **kw)
    # a tensor of its version: a backward pass that saved the pages would raise
    version = pages.data._version
    append()
    assert pages.data._version == version + 1


def test_in_a_graph(gpu):
    """A step captured once and replayed: append, read and attend, over changed inputs, with eager calls between."""
    dtype, kv, d = torch.bfloat16, 2, 128
    pages, table, k, v, positions, sequences = packed([2000, 500], 16, kv, d, d, dtype, seed=14, capacity=2100)
    eager, same, *_ = packed([2000, 500], 16, kv, d, d, dtype, seed=14, capacity=2100)
    rope = certex.Rotary(d)
    new_k, new_v, q = rand(2, kv, d, dtype=dtype), rand(2, kv, d, dtype=dtype), rand(2, 8, d, dtype=dtype)
    lens = ints([2000, 500])

    def step(p):
        p.append(new_k, new_v, table, lens, rotary=rope)
        return p.attend(q, table, lens + 1, window=1500), *p.read(table, lens)

    step(pages), step(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(pages)
    for i in range(3):
        lens += 1
        for x in (new_k, new_v, q):
            x.copy_(rand(*x.shape, dtype=dtype, seed=20 + i))
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        for x, y in zip(got, step(eager)):
            assert torch.equal(x, y)
