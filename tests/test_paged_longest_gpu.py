"""A sequence as long as a page table can be: 2^31 - 8 positions."""

import pytest
import torch

import libcertex_amd as certex
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_longest_sequence(gpu, dtype):
    """Appended to, attended over and selected from at its last positions; what would lie behind them does not count."""
    page, n, kv, d = 8, 2**31 - 8, 2, 16
    table = torch.zeros((1, n // page), dtype=torch.int32, device="cuda")
    table[0, -6:] = torch.tensor([3, 1, 5, 2, 6, 4], dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randn((48 if h == kv else 1, h, d), generator=g, device="cuda").to(dtype) for h in (kv, kv, 4))
    kp, vp = (torch.full((7, page, kv, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    at = torch.arange(n - 48, n, device="cuda", dtype=torch.int64)
    certex.append_pages(k, v, kp, vp, table, at, sequences=torch.zeros(48, dtype=torch.int32, device="cuda"))
    assert torch.equal(kp[4], k[40:]) and torch.equal(vp[3], v[:8])
    for short in (0, 1, 8):
        for window in (1, 7, 8, 20, 33):
            out, lse = certex.paged_attention(q, kp, vp, table, torch.tensor([n - short], device="cuda"), window=window,
                                              return_lse=True)
            seen = slice(48 - short - window, 48 - short)
            want, want_lse, spread, dots = ref.attend(q[0], k[seen], v[seen], d**-0.5)
            ref.assert_attended(out[0], want, spread, dots, window, d, lse[0], want_lse)
    scores = torch.randn((4, 1, 48), generator=g, device="cuda")
    out = certex.selected_attention(scores, at.expand(4, 1, 48).contiguous(), vp, 0.5, page_table=table[0])
    w = torch.softmax(0.5 * scores[:, 0].double().cpu(), -1)
    for h in range(4):
        rows = v[:, h // 2].double().cpu()
        ref.assert_attended(out[h], (w[h] @ rows)[None], (w[h] @ rows.abs())[None], scores[h].abs().max()[None].double().cpu(), 48, 1)
