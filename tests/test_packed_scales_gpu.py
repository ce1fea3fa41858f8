"""4-bit attention where the scales of a record differ: NaN beside others, steep ones beside flat ones."""

import pytest
import torch

import libcertex_amd as certex
from tests import packed_reference as pack
from tests import shaped_reference as ref
from tests.test_packed_gpu import TYPES, weight_unit
from tests.test_paged_gpu import ints, rand

pytestmark = pytest.mark.gpu


def check_columns(k, v, q, columns):
    """One sequence of all positions of k and v (n, kv, d): the other columns of the output are NaN, these as defined."""
    n, kv, d = k.shape
    pages = certex.PackedPages(-(-n // 16), 16, kv, d)
    table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda").flip(0)[None]
    positions = torch.arange(n, device="cuda")
    pages.append(k, v, table, positions, sequences=torch.zeros_like(positions))
    out, lse = pages.attend(q, table, ints([n]), return_lse=True)
    (keys, key_sizes), (values, value_sizes) = pack.stored(k), pack.stored(v)
    want = ref.attend(q, torch.tensor([n - 1]), keys, values[..., columns], d**-0.5, weight=weight_unit(q.dtype), key_sizes=key_sizes,
                      value_sizes=value_sizes[..., columns])
    ref.check(out[..., columns].contiguous(), lse, want)
    rest = torch.ones(d, dtype=torch.bool)
    rest[columns] = False
    assert out[..., rest.cuda()].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("n", [1, 2, 33, 34, 65, 97, 130])
def test_nan_beside_other_groups(gpu, dtype, d, n):
    """NaN in 64 elements of a value makes these columns NaN and no others, also where few positions are weighed with it."""
    for group in range(d // 64):
        k, v, q = rand(n, 2, d, dtype=dtype), rand(n, 2, d, dtype=dtype, seed=1), rand(1, 4, d, dtype=dtype, seed=2)
        v[n - 1, :, 64 * group + 5] = float("nan")
        columns = torch.arange(d)[torch.arange(d) // 64 != group]
        check_columns(k, v, q, columns)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nan, steep", [(0, 2), (1, 3), (6, 4), (12, 14), (20, 16)])
def test_nan_hides_no_steep_scale(gpu, dtype, nan, steep):
    """A scale a hundred and ten thousand times the others', in a record whose scales have a NaN among them."""
    for times in (100.0, 10_000.0):
        k, v, q = rand(40, 1, 128, dtype=dtype), rand(40, 1, 128, dtype=dtype, seed=1), rand(1, 4, 128, dtype=dtype, seed=2)
        v[steep, :, 64:] *= times
        v[nan, :, 3] = float("nan")
        check_columns(k, v, q, torch.arange(64, 128))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low, tiny, code", [
    (-6.5, 2.0**-60, 7), (-6.5, -(2.0**-60), 6), (-6.5, 2.0**-120, 7), (-6.5, 0.0, 6), (-7.5, -(2.0**-60), 7), (-7.5, 2.0**-60, 8),
    (-7.5, 0.0, 8), (-0.5, 2.0**-60, 1), (-14.5, -(2.0**-60), 14)])
def test_codes_next_to_a_tie(gpu, dtype, low, tiny, code):
    """Elements from `low` to low + 15, of scale 1: one next to 0 is past the middle of two codes by less than 64 bits hold of the
    distance from the offset."""
    x = torch.linspace(low, low + 15, 16).repeat(4)
    x[20] = tiny
    pages = certex.PackedPages(1, 8, 1, 64)
    k = x.to(dtype).cuda()[None, None]
    assert float(k[0, 0, 20]) == tiny
    table, position = ints([[0]]), ints([3])
    pages.append(k, k, table, position)
    for side in pages.read(table, position, dtype=torch.float32):
        want = x.clone()
        want[20] = low + code
        assert torch.equal(side[0, 0].cpu(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 192, 40])
@pytest.mark.parametrize("n", [7, 33, 120])
def test_weights_enter_whole(gpu, dtype, d, n):
    """Outputs of every type are as far off as float32 sums of them, however small they are beside the values: weights times scales
    meet the codes as two elements of 11 bits, the second cut (2^-21 of them at most), after one product (2^-24). Queries of 0 and slopes:
    the scores are nearly exact, so that little else is off, and among the outputs of many heads some are near 0."""
    heads = 64
    k, v = rand(n, 2, d, dtype=dtype), rand(n, 2, d, dtype=dtype, seed=1)
    q, slopes = torch.zeros(1, heads, d, dtype=dtype, device="cuda"), torch.linspace(0.001, 0.1, heads, device="cuda")
    pages = certex.PackedPages(-(-n // 16), 16, 2, d)
    table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda").flip(0)[None]
    positions = torch.arange(n, device="cuda")
    pages.append(k, v, table, positions, sequences=torch.zeros_like(positions))
    out, lse = pages.attend(q, table, ints([n]), return_lse=True, slopes=slopes)
    (keys, key_sizes), (values, value_sizes) = pack.stored(k), pack.stored(v)
    ref.check(out, lse, ref.attend(q, torch.tensor([n - 1]), keys, values, d**-0.5, weight=2.0**-21 + 2.0**-24, key_sizes=key_sizes,
                                   value_sizes=value_sizes, slopes=slopes))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256, 80])
def test_scores_are_float32_sums(gpu, dtype, d):
    """Scores, which the float32 logarithms show where a sequence has one position, are off as float32 sums of their terms in any order
    are, as random roundings: u sum |scale q k| / sqrt(d) in the mean over dimensions and 8 u of the terms' own, 4 times that at most, and
    8 u of the logarithm itself. Products of codes as numbers of 4 bits only would keep no such sums."""
    heads = 64
    k, v, q = rand(1, 1, d, dtype=dtype), rand(1, 1, d, dtype=dtype, seed=1), rand(1, heads, d, dtype=dtype, seed=2)
    pages = certex.PackedPages(1, 8, 1, d)
    table, zero = ints([[0]]), ints([0])
    pages.append(k, v, table, zero)
    lse = pages.attend(q, table, ints([1]), return_lse=True)[1]
    held, sizes = pack.stored(k)
    want = (q[0].double().cpu() @ held[0, 0]) * d**-0.5
    size = float((q[0].double().cpu().abs() @ sizes[0, 0]).max()) * d**-0.5
    u = 2.0**-24
    assert float((lse[0].double().cpu() - want).abs().max()) <= 4 * (size / d**0.5 + 8) * u + 8 * u * float(want.abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [128, 192, 256, 96])
@pytest.mark.parametrize("high, low", [(1.0, 2.0**-10), (2.0**-10, 1.0), (2.0**12, 2.0**-8), (2.0**-8, 2.0**12)])
def test_groups_of_different_sizes(gpu, dtype, d, high, low):
    """Values of one group of 64 elements are as precise as if the others were not there, though those are up to 2^20 times as large: as in
    test_weights_enter_whole, for each group by itself."""
    n, heads = 40, 32
    k, v = rand(n, 2, d, dtype=dtype), rand(n, 2, d, dtype=dtype, seed=1)
    for group in range(-(-d // 64)):
        v[..., 64 * group : 64 * group + 64] *= high if group % 2 == 0 else low
    q, slopes = torch.zeros(1, heads, d, dtype=dtype, device="cuda"), torch.linspace(0.001, 0.1, heads, device="cuda")
    pages = certex.PackedPages(-(-n // 16), 16, 2, d)
    table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda").flip(0)[None]
    positions = torch.arange(n, device="cuda")
    pages.append(k, v, table, positions, sequences=torch.zeros_like(positions))
    out, lse = pages.attend(q, table, ints([n]), return_lse=True, slopes=slopes)
    (keys, key_sizes), (values, value_sizes) = pack.stored(k), pack.stored(v)
    ref.check(out, lse, ref.attend(q, torch.tensor([n - 1]), keys, values, d**-0.5, weight=2.0**-21 + 2.0**-24, key_sizes=key_sizes,
                                   value_sizes=value_sizes, slopes=slopes))
