"""The attention operators' plans at the sizes where they change: more sequences than a wave has lanes, half as many shares,
ids by ranges over pages and over the most ranges, gradients of every type."""

import pytest
import torch

import libcertex_amd as certex
from tests import paged_reference as ref
from tests.test_paged_gpu import TYPES, check_attend, check_selected, paged, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [64, 65, 130, 200])
def test_many_sequences(gpu, dtype, n):
    """Lengths are read 64 at a time: sequences on both sides of every 64th, some without a position."""
    lens = [(37 * i) % 300 + 1 for i in range(n)]
    for i in (0, 62, 63, 64, 65, 127, 128, 129, 191, n - 1):
        if i < n:
            lens[i] = 0
    check_attend(lens, 4, 2, 64, 64, 16, dtype, seed=20)
    check_attend([0] * (n - 1) + [500], 4, 2, 64, 64, 16, dtype, seed=21)
    check_attend([500] + [0] * (n - 1), 4, 2, 64, 64, 16, dtype, window=300, seed=22)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[9000, 70, 0, 8000], [17_000], [9000, 0, 7000]])
def test_half_the_shares(gpu, dtype, lens):
    """64 key heads of 128 take 8 shares each, and 4 from 128 tiles of 128 positions on (135 and 133 here, 126 in the last):
    the sequences are cut elsewhere."""
    check_attend(lens, 64, 64, 128, 128, 64, dtype, seed=23)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [7, 64])
def test_selected_ranges_of_pages(gpu, dtype, page):
    """Ids taken by ranges of rows, whose values lie in the pages of a shuffled table; pages are missing."""
    n, heads, kv, m, k, dv = 35_000, 4, 2, 64, 2048, 128
    _, vp, table, _, values = paged([n], page, kv, 8, dv, dtype, seed=24)
    scores, ids = rand(heads, m, k, scale=5.0), torch.randint(0, n, (heads, m, k), device="cuda")
    table = table[0].contiguous()
    host = values[0].double().cpu()
    few = [0, 1, m - 1]
    out, lse = certex.selected_attention(scores, ids, vp, 0.3, page_table=table, return_lse=True)
    check_selected(scores[:, few], ids[:, few], lambda g: host[:, g], heads, kv, 0.3, out[:, few], lse[:, few])
    gone = torch.zeros_like(table, dtype=torch.bool)
    gone[::5], gone[-1], gone[3:40] = True, True, True
    table[gone] = torch.where(torch.arange(int(gone.sum()), device="cuda") % 2 == 0, -1, vp.shape[0]).int()
    out, lse = certex.selected_attention(scores, ids, vp, 0.3, page_table=table, return_lse=True)
    left = torch.where(gone[ids // page], -1, ids)
    check_selected(scores[:, few], left[:, few], lambda g: host[:, g], heads, kv, 0.3, out[:, few], lse[:, few])


def test_selected_most_ranges(gpu):
    """Values of 64 ranges and more (138 MB a head): the last of them ends where the ids do."""
    n, heads, m, k, dv = 270_000, 4, 100, 2048, 128
    values, scores = rand(1, n, dv), rand(heads, m, k, scale=5.0)
    ids = torch.randint(0, n, (heads, m, k), device="cuda")
    ids[0, 0] = n - 1
    ids[0, 1] = torch.arange(n - k, n, device="cuda")
    ids[0, 2] = -1
    ids[0, 3, 5:] = n
    ids[0, 4] = torch.arange(k, device="cuda")
    out, lse = certex.selected_attention(scores, ids, values, 0.3, return_lse=True)
    host = values.double().cpu()
    few = [0, 1, 2, 3, 4, m - 1]
    check_selected(scores[:1, few], ids[:1, few], lambda g: host[g], 1, 1, 0.3, out[:1, few], lse[:1, few])
    check_selected(scores[3:, few], ids[3:, few], lambda g: host[g], 1, 1, 0.3, out[3:, few], lse[3:, few])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d, r", [(64, 48), (61, 34)])
def test_rotation_gradient_of_every_type(gpu, dtype, layout, d, r):
    """Through strided inputs and broadcast gradients; what is not turned passes bit for bit, both ways."""
    rope = certex.Rotary(d, rotary_dim=r, layout=layout)
    p = torch.arange(30, device="cuda") * 1009
    wide, dy = rand(30, 3, d + 9, dtype=dtype), rand(30, 3, d + 9, dtype=dtype, seed=1)
    for lo in (0, 3):
        x = wide[..., lo : lo + d].detach().requires_grad_()
        y = rope(x, p)
        ref.assert_rotated(y.detach(), x.detach(), ref.rotate(x.detach(), p, rope.frequencies, layout, r), layout, r)
        assert torch.equal(y[..., r:], x[..., r:])
        for g in (dy[..., lo : lo + d], dy[..., :1].expand(30, 3, d), dy[:1, :1, :d].expand(30, 3, d)):
            (dx,) = torch.autograd.grad(y, x, g, retain_graph=True)
            ref.assert_rotated(dx, g, ref.rotate(g, p, rope.frequencies, layout, r, transpose=True), layout, r)
            assert dx.dtype == dtype and torch.equal(dx[..., r:], g[..., r:])
