"""Attention of prompts where page tables have rows without new tokens, and calls that split the positions of many sequences."""

import pytest
import torch

import libcertex_amd as certex
from tests import shaped_reference as ref
from tests.test_paged_gpu import ints, paged, rand
from tests.test_prompt_gpu import TYPES, check_prompt, slopes_of, weight_unit

pytestmark = pytest.mark.gpu


def idle(news, rows, at, rest=0):
    """`rows` numbers: those of `news` at the rows `at`, and `rest` elsewhere."""
    out = [rest] * rows
    for n, s in zip(news, at):
        out[s] = n
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 64, 65, 256, 257, 1000])
def test_idle_rows(gpu, dtype, rows):
    """A few tokens of a few sequences, the first and the last row among them: positions are split and joined."""
    at = sorted({0, 1, rows // 3, rows - 1})
    news = idle([16, 1, 3, 40][: len(at)], rows, at)
    pasts = idle([2_000, 700, 0, 300][: len(at)], rows, at, rest=5)
    check_prompt(news, pasts, 8, 2, 128, 128, 64, dtype, seed=70)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, where", [(70, 0), (70, 69), (300, 255), (300, 256), (1025, 1024)])
def test_one_busy_row(gpu, dtype, rows, where):
    """All tokens are of one row of many: as many splits as it would have alone, and the same bits."""
    past, n, heads = 3_000, 20, 8
    kp, vp, table, keys, values = paged([past + n], 16, 2, 64, 64, dtype, seed=71)
    q = rand(n, heads, 64, dtype=dtype)
    alone, alone_lse = certex.prompt_attention(q, kp, vp, table, ints([past + n]), ints([0, n]), return_lse=True)
    many = torch.full((rows, table.shape[1]), -1, dtype=torch.int32, device="cuda")
    many[where] = table[0]
    first = ints([0] * (where + 1) + [n] * (rows - where))
    out, lse = certex.prompt_attention(q, kp, vp, many, ints(idle([past + n], rows, [where], rest=9)), first, return_lse=True)
    assert torch.equal(out, alone) and torch.equal(lse, alone_lse)
    ref.check(out, lse, ref.attend(q, torch.arange(past, past + n), keys[0], values[0], 64**-0.5, weight=weight_unit(dtype)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sequences", [40, 64, 65, 100, 300])
def test_short_sequences_over_split_caches(gpu, dtype, sequences):
    """One token and a few of each of many sequences, with bent scores, a window and prefixes too: few enough to be split, and so many
    that they are not."""
    g = torch.Generator().manual_seed(72)
    news = torch.randint(0, 3, (sequences,), generator=g).tolist()
    pasts = torch.randint(0, 1_500, (sequences,), generator=g).tolist()
    pasts[0], news[0], news[-1] = 2_500, 1, 2
    check_prompt(news, pasts, 2, 1, 64, 64, 16, dtype, seed=73)
    check_prompt(news, pasts, 4, 2, 128, 40, 16, dtype, window=900, cap=20.0, slopes=slopes_of(4),
                 prefix=[i % 50 for i in range(sequences)], seed=74)


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_heads_of_many_sequences(gpu, dtype):
    """Two workgroups share a row's columns and several its positions."""
    news, pasts = [1, 2, 0, 5] + [0] * 70 + [1], [1_200, 30, 900, 2_000] + [4] * 70 + [600]
    check_prompt(news, pasts, 4, 2, 256, 200, 16, dtype, seed=75)


def test_workspace_is_enough(gpu):
    """The kernels write no further than the workspace that the query names, however the tokens lie in the sequences: bytes behind
    it stay as they were."""
    import ctypes

    from libcertex_amd import _capi as C
    from tests.test_paged import _tensor

    dtype, kv, heads, d, page, width = torch.bfloat16, 2, 8, 64, 16, 130
    n_pages, tokens, rows = 200, 40, 90
    q, pool = rand(tokens, heads, d, dtype=dtype), rand(n_pages, page, kv, d, dtype=dtype)
    table = torch.randint(0, n_pages, (rows, width), generator=torch.Generator().manual_seed(1)).int().cuda()
    lens = ints([page * width] * rows)

    def view(t):
        m = _tensor(tuple(t.shape), t.dtype)
        m.dl_tensor.data = t.data_ptr()
        return m

    out = torch.empty(tokens, heads, d, dtype=dtype, device="cuda")
    bytes_ = ctypes.c_int64()
    qv, kv_, tv, lv, ov = (view(t) for t in (q, pool, table, lens, out))
    C.check(C.lib().cuvsCertexPromptAttentionWorkspace(*[ctypes.addressof(x) for x in (qv, kv_, kv_, tv)], 0, ctypes.byref(bytes_)))
    assert bytes_.value > 0
    for news in ([tokens] + [0] * (rows - 1), [0] * (rows - 1) + [tokens], [1] * tokens + [0] * (rows - tokens), [0, 1] * 40 + [0] * 10,
                 [0, 8, 8, 8, 8, 8] + [0] * (rows - 6)):
        first = ints([sum(news[:s]) for s in range(rows + 1)])
        work = torch.full((bytes_.value + (1 << 20),), 0x5A, dtype=torch.uint8, device="cuda")
        fv, wv = view(first), view(work)
        wv.dl_tensor.shape[0] = bytes_.value
        C.check(C.lib().cuvsCertexPromptAttention(C.stream_resources(), *[ctypes.addressof(x) for x in (qv, kv_, kv_, tv, lv, fv)], None,
                                                  d**-0.5, 0.0, None, 0, ctypes.addressof(wv), ctypes.addressof(ov), None))
        torch.cuda.synchronize()
        assert (work[bytes_.value :] == 0x5A).all()
        assert torch.equal(out, certex.prompt_attention(q, pool, pool, table, lens, first))


@pytest.mark.parametrize("window", [2**31, 2**32 + 1, 2**63 - 129, 2**63 - 1])
def test_windows_past_all_positions(gpu, window):
    """A window that holds every position is none, also of tokens before position 0."""
    dtype = torch.bfloat16
    kp, vp, table, keys, values = paged([40, 600], 16, 2, 64, 64, dtype, seed=76)
    q, lens, first = rand(250, 4, 64, dtype=dtype), ints([40, 600]), ints([0, 200, 250])
    want = certex.prompt_attention(q, kp, vp, table, lens, first, return_lse=True)
    for got, x in zip(certex.prompt_attention(q, kp, vp, table, lens, first, window=window, return_lse=True), want):
        assert torch.equal(got, x)
    ref.check(want[0][160:200], want[1][160:200], ref.attend(q[160:200], torch.arange(40), keys[0], values[0], 0.125,
                                                             weight=weight_unit(dtype)))
    one = q[:2].contiguous()
    assert torch.equal(certex.paged_attention(one, kp, vp, table, lens, window=window), certex.paged_attention(one, kp, vp, table, lens))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 192, 256, 40])
@pytest.mark.parametrize("n, past", [(7, 0), (33, 0), (20, 100), (3, 1_500)])
def test_weights_enter_whole(gpu, dtype, d, n, past):
    """Outputs of 16-bit types are nearly as far off as float32 sums of their values, however small they are beside these: a weight is the
    sum of two elements of the type, each the nearest, so that it is off by the square of the type's half unit (and float32's). Queries
    of 0 and slopes: the scores are nearly exact, so that little else is off, and among the outputs of many heads some are near 0."""
    heads = 16
    slopes = torch.linspace(0.001, 0.1, heads, device="cuda")
    kp, vp, table, keys, values = paged([past + n], 16, 2, d, d, dtype, seed=77)
    q = torch.zeros(n, heads, d, dtype=dtype, device="cuda")
    out, lse = certex.prompt_attention(q, kp, vp, table, ints([past + n]), ints([0, n]), slopes=slopes, return_lse=True)
    weight = 0.0 if dtype == torch.float32 else weight_unit(dtype) ** 2
    ref.check(out, lse, ref.attend(q, torch.arange(past, past + n), keys[0], values[0], d**-0.5, slopes=slopes, weight=weight))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [8, 64, 70, 300])
def test_prompts_beside_single_tokens(gpu, dtype, rows):
    """A piece of a prompt behind a long cache beside single tokens of short ones: the long one alone is split. Lengths of 0 and below the
    tokens among them, and calls of nothing else."""
    g = torch.Generator().manual_seed(78)
    news = [70, 1, 1, 1, 0, 1, 1, 1] + [int(torch.randint(0, 2, (1,), generator=g)) for _ in range(rows - 8)]
    pasts = [6_000, 100, 40, 0, 9, 300, 2_000, 5] + [int(torch.randint(0, 90, (1,), generator=g)) for _ in range(rows - 8)]
    check_prompt(news, pasts, 4, 1, 64, 64, 16, dtype, seed=79)
    kp, vp, table, *_ = paged([200] * rows, 16, 1, 64, 64, dtype, seed=80)
    q, first = rand(2 * rows, 4, 64, dtype=dtype), ints([2 * i for i in range(rows + 1)])
    out, lse = certex.prompt_attention(q, kp, vp, table, ints([0] * rows), first, return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()
    out, lse = certex.prompt_attention(q, kp, vp, table, ints([1, 200] * (rows // 2)), first, return_lse=True)
    assert (out[0::4] == 0).all() and (lse[0::4] == float("-inf")).all() and lse[1::4].isfinite().all() and lse[2::4].isfinite().all()
