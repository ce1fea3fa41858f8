"""The prompt, bent and 4-bit attention operators without a GPU: refusals of the Python functions and of the C entry points."""

import ctypes

import pytest
import torch

import libcertex_amd as certex
from libcertex_amd import _capi as C
from tests.test_paged import _need, _tensor


def _prompt(q=(20, 8, 64), k=(4, 16, 2, 64), v=(4, 16, 2, 64), table=(2, 2), dtype=torch.float16, k_type=None, window=0,
            table_type=torch.int32, device=C.kDLROCM, strides=None):
    t = [_tensor(q, dtype, device), _tensor(k, k_type or dtype, strides=strides), _tensor(v, dtype), _tensor(table, table_type)]
    out = ctypes.c_int64()
    C.check(C.lib().cuvsCertexPromptAttentionWorkspace(*[ctypes.addressof(x) for x in t], window, ctypes.byref(out)))
    return out.value


def test_prompt_checks():
    """The checks that the call and its workspace query share need no device."""
    assert _prompt() >= 0 and _prompt(q=(1, 6, 33), k=(4, 8, 3, 33), v=(4, 8, 3, 256)) >= 0
    assert _prompt(table=(0, 2)) >= 0 and _prompt(q=(0, 8, 64)) >= 0
    assert _prompt(q=(8192, 32, 64), k=(4, 16, 8, 64), v=(4, 16, 8, 64), table=(1, 128)) == 0  # fills the chip without splits
    assert _prompt(q=(1, 32, 64), k=(4, 64, 8, 64), v=(4, 64, 8, 64), table=(1, 2048)) > 0
    for kw, match in [
        (dict(q=(20, 8, 63)), "same head dimension"), (dict(q=(20, 7, 64)), "multiple of the key heads"),
        (dict(k=(4, 12, 2, 64), v=(4, 12, 2, 64)), "multiple of 8"), (dict(v=(4, 8, 2, 64)), "v_pages must have shape"),
        (dict(v=(4, 16, 2, 257)), "between 1 and 256"), (dict(q=(20, 8, 272), k=(4, 16, 2, 272)), "between 1 and 256"),
        (dict(k_type=torch.bfloat16), "element type"), (dict(dtype=torch.int32), "float32, float16 or bfloat16"),
        (dict(table_type=torch.int64), "must be int32"), (dict(device=C.kDLCPU), "device memory"), (dict(window=-1), "window"),
        (dict(q=(20, 8, 64, 1)), "3 dimensions"), (dict(strides=(2048, 128, 64, 2)), "dense in its last dimension"),
        (dict(table=(70_000, 2)), "65535 sequences"), (dict(table=(2, 1 << 27)), "2\\^31"), (dict(q=(1 << 30, 8, 64)), "too many tokens"),
        (dict(q=(1 << 27, 8, 64)), "too many tokens"),
    ]:
        with pytest.raises(ValueError, match=match):
            _prompt(**kw)
    # the last positions below 2^31 of a page table are refused, not those before
    assert _prompt(k=(4, 64, 2, 64), v=(4, 64, 2, 64), table=(1, (1 << 25) - 1)) >= 0
    with pytest.raises(ValueError, match="at most 2\\^31 - 64 positions"):
        _prompt(k=(4, 8, 2, 64), v=(4, 8, 2, 64), table=(1, (1 << 28) - 7))


def _record(dim, vdim):
    out = ctypes.c_int64()
    C.check(C.lib().cuvsCertexPackedRecord(dim, vdim, ctypes.byref(out)))
    return out.value


def test_packed_records():
    """8 positions: half a byte for each of the padded dimensions, 4 bytes for each 64 of them, on both sides."""
    padded = {1: 64, 64: 64, 65: 96, 96: 96, 97: 128, 128: 128, 129: 192, 192: 192, 193: 256, 256: 256}
    for d, p in padded.items():
        for dv, pv in padded.items():
            assert _record(d, dv) == 8 * ((p + pv) // 2 + 4 * (-(-p // 64) + -(-pv // 64)))
    for bad in ((0, 64), (64, 0), (257, 64), (64, 257), (-1, 64)):
        with pytest.raises(ValueError, match="between 1 and 256"):
            _record(*bad)


def _packed(q=(2, 8, 64), pages=(4, 2, 2, 576), vdim=64, table=(2, 2), dtype=torch.float16, page_type=torch.uint8, window=0,
            table_type=torch.int32, offset=0):
    t = [_tensor(q, dtype), _tensor(pages, page_type), _tensor(table, table_type)]
    t[1].dl_tensor.byte_offset = offset
    out = ctypes.c_int64()
    C.check(C.lib().cuvsCertexPackedAttentionWorkspace(ctypes.addressof(t[0]), ctypes.addressof(t[1]), vdim,
                                                       ctypes.addressof(t[2]), window, ctypes.byref(out)))
    return out.value


def test_packed_checks():
    assert _packed() == 0 and _packed(table=(2, 2000)) > 0 and _packed(dtype=torch.float32) == 0
    for kw, match in [
        (dict(q=(2, 7, 64)), "multiple of the key heads"), (dict(q=(3, 8, 64)), "one row per sequence"),
        (dict(q=(2, 8, 65)), "records of 736 bytes"), (dict(vdim=128), "records of 864 bytes"), (dict(vdim=0), "between 1 and 256"),
        (dict(q=(2, 8, 257)), "between 1 and 256"), (dict(pages=(4, 2, 2, 577)), "records of 576 bytes"),
        (dict(pages=(4, 0, 2, 576)), "heads"), (dict(pages=(4, 2, 0, 576)), "multiple of 8"), (dict(pages=(4, 2, 576)), "4 dimensions"),
        (dict(page_type=torch.float16), "uint8"), (dict(dtype=torch.int64), "float32, float16 or bfloat16"),
        (dict(table_type=torch.int64), "must be int32"), (dict(window=-1), "window"), (dict(offset=8), "aligned to 16 bytes"),
        (dict(table=(2, 1 << 28)), "fewer than 2\\^31"), (dict(q=(2, 8, 64, 1)), "3 dimensions"),
    ]:
        with pytest.raises(ValueError, match=match):
            _packed(**kw)


def test_null_arguments_are_errors():
    L = C.lib()
    n = ctypes.c_int64()
    with pytest.raises(ValueError, match="q is NULL"):
        C.check(L.cuvsCertexPromptAttentionWorkspace(None, None, None, None, 0, ctypes.byref(n)))
    with pytest.raises(ValueError, match="q is NULL"):
        C.check(L.cuvsCertexPackedAttentionWorkspace(None, None, 64, None, 0, ctypes.byref(n)))
    for call in [lambda: L.cuvsCertexPackedRecord(64, 64, None), lambda: L.cuvsCertexPromptAttentionWorkspace(*[None] * 4, 0, None),
                 lambda: L.cuvsCertexPackedAttentionWorkspace(None, None, 64, None, 0, None)]:
        with pytest.raises(ValueError, match="NULL"):
            C.check(call())
    for call in [lambda: L.cuvsCertexPromptAttention(0, *[None] * 7, 1.0, 0.0, None, 0, *[None] * 3),
                 lambda: L.cuvsCertexPagedAttentionShaped(0, *[None] * 5, 1.0, 0.0, None, 0, *[None] * 3),
                 lambda: L.cuvsCertexPackPages(0, 0, *[None] * 6), lambda: L.cuvsCertexUnpackPages(0, *[None] * 6),
                 lambda: L.cuvsCertexPackedAttention(0, None, None, 64, None, None, 1.0, 0.0, None, 0, *[None] * 3)]:
        with pytest.raises(ValueError, match="resources handle is NULL"):
            C.check(call())


def test_host_tensors_are_refused():
    x, i = torch.zeros(3, 2, 8), torch.zeros(3, dtype=torch.int32)
    pool, table = torch.zeros(2, 8, 2, 8), torch.zeros(3, 2, dtype=torch.int32)
    for call in [lambda: certex.prompt_attention(x, pool, pool, table, i, torch.zeros(4, dtype=torch.int32)),
                 lambda: certex.paged_attention(x, pool, pool, table, i, cap=5.0),
                 lambda: certex.PackedPages(2, 8, 2, 8, data=torch.zeros(2, 2, 1, 576, dtype=torch.uint8))]:
        with pytest.raises(ValueError, match="GPU"):
            call()
    for bad in (dict(page_size=12), dict(page_size=0), dict(n_pages=-1), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=257),
                dict(value_dim=300)):
        with pytest.raises(ValueError):
            certex.PackedPages(**{**dict(n_pages=2, page_size=8, n_kv_heads=2, head_dim=64), **bad})


@pytest.mark.parametrize("tokens, heads, kv, rows, positions, most", [
    (16, 32, 8, 64, 16_384, 20), (16, 32, 8, 256, 16_384, 20), (64, 32, 8, 64, 16_384, 40), (1_000, 8, 8, 1_000, 4_096, 40),
    (1, 64, 8, 1_024, 131_072, 20), (8, 32, 8, 4_096, 32_768, 20), (128, 32, 32, 128, 8_192, 40), (1, 8, 8, 65_535, 32_704, 1),
    (2_000, 32, 8, 2_000, 32_768, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_workspace_is_of_the_tokens(tokens, heads, kv, rows, positions, most, dtype, d):
    """Few tokens in tables of many rows: MB of partials (heads of 128; in proportion to the dimension), a row for each token, head and
    split, whatever rows the table has."""
    pool = (4, 64, kv, d)
    got = _prompt(q=(tokens, heads, d), k=pool, v=pool, table=(rows, positions // 64), dtype=dtype)
    # (heads of 64 run three workgroups per compute unit, those of 128 two)
    assert got <= most * 1e6 * max(1.0, (d + 2) / 128) * 1.5
    assert got == _prompt(q=(tokens, heads, d), k=pool, v=pool, table=(1, positions // 64), dtype=dtype)


def test_prompt_tables_of_any_rows():
    """What a call may launch goes by its tokens: a table of the most rows is no reason to refuse one."""
    assert _prompt(q=(1, 256, 64), k=(4, 16, 256, 64), v=(4, 16, 256, 64), table=(65_535, 2)) >= 0


@pytest.mark.parametrize("window", [2**31, 2**32 + 1, 2**63 - 129, 2**63 - 1])
def test_windows_past_all_positions(window):
    """A window that holds every position is none: the same splits and shares, whatever is added to it."""
    few = dict(q=(1, 32, 64), k=(4, 64, 8, 64), v=(4, 64, 8, 64), table=(1, 2048))
    assert _prompt(**few, window=window) == _prompt(**few) > 0
    assert _packed(table=(2, 2000), window=window) == _packed(table=(2, 2000)) > 0
    assert _need(table=(2, 2000), window=window) == _need(table=(2, 2000)) > 0
