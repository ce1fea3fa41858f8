"""KeyCache.attend takes the values of its own keys: of its heads, and of every key. It has no gradient, and says so."""

import pytest
import torch

import libcertex_amd as certex

pytestmark = pytest.mark.gpu


def test_values_of_other_keys_are_refused(gpu):
    g = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

    cache = certex.KeyCache(4, 64, k=20).append(rand(4, 100, 64))
    q, values = rand(8, 3, 64), rand(4, 100, 32)
    pages, table = rand(9, 16, 4, 32), torch.arange(7, dtype=torch.int32, device="cuda")
    good = cache.attend(q, values)
    for call, match in [
        (lambda: cache.attend(q, values[:, :99]), "100 keys, not 99"), (lambda: cache.attend(q, values[:2]), "4 heads, not 2"),
        (lambda: cache.attend(q, values[:1].expand(8, 100, 32)), "4 heads, not 8"),
        (lambda: cache.attend(q, pages, page_table=table[:6]), "100 keys, not 96"),
        (lambda: cache.attend(q, pages[:, :, :2], page_table=table), "4 heads, not 2"),
        (lambda: cache.attend(q, pages), "3 dimensions"), (lambda: cache.attend(q, values, page_table=table), "4 dimensions"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    more = torch.cat([values, rand(4, 50, 32)], 1)  # room for keys to come
    assert torch.equal(cache.attend(q, more), good)
    flat = pages[:7].reshape(112, 4, 32)[:100].transpose(0, 1)
    assert torch.equal(cache.attend(q, pages, page_table=table), cache.attend(q, flat))
    missing = table.clone()
    missing[2] = -1  # a page that is gone does not count, as ever
    assert cache.attend(q, pages, page_table=missing).isfinite().all()


def test_differentiated_queries_are_refused(gpu):
    """A gradient or a tangent of the queries would be lost in the search: an error, as for the values."""
    import torch.autograd.forward_ad as fwd

    keys, q, values = (torch.randn(s, device="cuda") for s in ((2, 50, 64), (4, 3, 64), (2, 50, 32)))
    cache = certex.KeyCache(2, 64, k=20).append(keys)
    q.requires_grad_()
    for call in (lambda: cache.attend(q, values), lambda: cache.attend(q.detach(), values.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no gradient"):
            call()
    with torch.no_grad():
        want = cache.attend(q, values)
    q = q.detach()
    assert torch.equal(cache.attend(q, values), want) and torch.equal(cache.attend(q.cpu().numpy(), values), want)
    with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        cache.attend(fwd.make_dual(q, torch.ones_like(q)), values)
