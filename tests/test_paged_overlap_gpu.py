"""Calls whose output lies in part where they read are refused; what shares no element is taken, however near it lies."""

import pytest
import torch

import libcertex_amd as certex
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def rand(*shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d, r", [(64, 64), (61, 34), (128, 64)])
def test_partial_overlap_is_refused(gpu, layout, d, r):
    rope = certex.Rotary(d, rotary_dim=r, layout=layout)
    p = torch.arange(6, device="cuda")
    flat = rand(40 * 3 * d)

    def at(start, strides=None, shape=(6, 3, d)):
        return flat.as_strided(shape, strides or (3 * d, d, 1), start)

    before = flat.clone()
    for x, out in [
        (at(0), at(1)), (at(1), at(0)), (at(0), at(8)), (at(0), at(d)), (at(0), at(3 * d)), (at(7 * 3 * d), at(5 * 3 * d)),
        (at(0), at(0, (d, 6 * d, 1))),  # its own memory, tokens and heads transposed
        (at(0, (2 * 3 * d, d, 1)), at(2 * 3 * d - 1, (2 * 3 * d, d, 1))),  # alternate rows, one element off
        (at(0, (0, d, 1)), at(0)),  # one token for all
        (at(0), at(40, (3 * d + 1, d, 1))),
    ]:
        with pytest.raises(ValueError, match="must not share memory in part"):
            rope(x, p, out=out)
    for out in (at(0, (2 * d, d, 1)), at(0, (3 * d, d - 1, 1)), at(0, (d, d, 1))):  # rows that run into one another
        with pytest.raises(ValueError, match="none of its elements may share memory"):
            rope(at(20 * 3 * d), p, out=out)
    assert torch.equal(flat, before)
    for x, out in [(at(0), at(6 * 3 * d)), (at(0, (2 * 3 * d, d, 1)), at(3 * d, (2 * 3 * d, d, 1))), (at(5), at(5)),
                   (at(0, (6 * d, 2 * d, 1)), at(d, (6 * d, 2 * d, 1))),
                   (at(0, (6 * d, 0, 1)), at(d, (6 * d, d, 1)))]:  # a head of a row turned for three heads of it
        held = x.clone()
        want = rope(held, p)
        assert rope(x, p, out=out) is out and torch.equal(out, want)
        ref.assert_rotated(out, held, ref.rotate(held, p, rope.frequencies, layout, r), layout, r)


def test_pages_that_share_memory_with_themselves_are_refused(gpu):
    flat, table = torch.zeros(40_000, dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    x, p = rand(2, 2, 64), torch.arange(2, device="cuda")
    pool, good = flat.as_strided((3, 8, 2, 64), (1000, 128, 64, 1)), torch.zeros((3, 8, 2, 64), dtype=torch.bfloat16, device="cuda")
    for pages in ((pool, good), (good, pool)):
        with pytest.raises(ValueError, match="none of its elements may share memory"):
            certex.append_pages(x, x, *pages, table, p)
    assert (flat == 0).all() and (good == 0).all()
    both = torch.zeros((3, 8, 2, 128), dtype=torch.bfloat16, device="cuda")  # keys and values side by side
    certex.append_pages(x, 2 * x, both[..., :64], both[..., 64:], table, p)
    assert torch.equal(both[0, [0, 1]], torch.cat([x, 2 * x], -1)) and (both[0, 2:] == 0).all() and (both[1:] == 0).all()
