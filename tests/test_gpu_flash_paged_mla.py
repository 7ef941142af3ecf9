"""GPU parity of flash_paged_mla against softmax attention in 64 bits over the same pages.

Tolerance of an output element, from its roundings: the result to bf16 (2^-8 of it), every probability times key scale
to bf16 (2^-8 of sum_j p_j |latent_j|), and the scores' error e (their 576 products in fp32) and the exponential's, at
most 2 (e + 2^-18) of the same sum.  lse: e and a few units of fp32."""
import math

import pytest
import torch

from oracle import paged
from tests import _paged
from tilert_amd.flash_paged_mla import flash_paged_mla
from tilert_amd.flash_sparse_mla import softmax_scale

pytestmark = pytest.mark.gpu
SCALE = softmax_scale("deepseek_v3_2")


def run(cuda, q, qp, pages, table, cu, lens, **kw):
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=cuda)
    lse = torch.full(q.shape[:-1], 7.0, device=cuda)
    flash_paged_mla(*_paged.to(cuda, q, qp, pages, table, cu, lens), out, lse, model_arch="deepseek_v3_2", **kw)
    torch.cuda.synchronize()
    return out, lse


def queries(rows, heads, seed, std=0.5):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(rows, heads, n, generator=g) * std).to(torch.bfloat16) for n in (512, 64)]


def check(cuda, q, qp, pages, table, cu, lens, out, lse, scale=SCALE):
    want, want_lse, spread, slack = paged.attention(*_paged.to(cuda, q, qp, pages, table, cu, lens), scale)
    mine = torch.zeros_like(want_lse, dtype=torch.bool)
    mine[:int(cu[-1])] = True
    bad = mine & torch.isnan(want_lse)  # the definition gives NaN: a NaN in a key that is seen
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    e = slack[..., None]
    tol = 2 ** -8 * want.abs() + (2 ** -8 + 2 * (e + 2 ** -18)) * spread
    off = (out.double() - want).abs()
    fine = mine & ~bad
    assert torch.all(off[fine] <= tol[fine]), (off[fine] / tol[fine].clamp_min(1e-30)).max()
    assert torch.all(out[~mine] == 7.0) and torch.all(lse[~mine] == 7.0)  # rows of no sequence
    seen = mine & torch.isfinite(want_lse)
    assert torch.all((lse.double() - want_lse).abs()[seen] <= (slack + 2 ** -20 * (1 + want_lse.abs()))[seen])
    assert torch.isneginf(lse[fine & ~seen]).all() and torch.all(out[fine & ~seen] == 0)


CASES = [  # new tokens, cache lengths, heads, padding
    ([1], [1], 16, 0), ([1], [2], 1, 0), ([1], [31], 16, 1), ([1], [32], 8, 0), ([1], [33], 16, 0), ([1], [64], 20, 0),
    ([1], [65], 16, 0), ([1], [129], 128, 0), ([1], [500], 10, 0), ([4], [4], 16, 0), ([4], [300], 16, 2),
    ([7], [70], 3, 0), ([33], [40], 16, 0), ([1], [4000], 16, 0), ([2], [5000], 128, 0), ([257], [700], 16, 5),
    ([64], [64], 20, 0), ([1, 1, 1], [10, 200, 64], 16, 0), ([1, 5, 0, 40, 1], [90, 5, 33, 400, 1], 16, 3),
    ([0, 0, 3], [0, 9, 64], 8, 1), ([1] * 70, list(range(1, 211, 3)), 16, 4), ([100, 1, 1], [130, 3000, 1], 20, 0),
    ([1] * 5, [64 * i for i in range(1, 6)], 128, 0), ([500], [1500], 8, 0), ([1], [40000], 16, 0), ([3], [30000], 8, 0),
    ([4], [30000], 16, 0), ([700, 300], [2000, 2500], 16, 0), ([1] * 40, [100 * i + 1 for i in range(40)], 16, 0),
]


@pytest.mark.parametrize("new,total,heads,pad", CASES)
def test_against_64_bits(cuda, new, total, heads, pad):
    print("case", new[:8], total[:8], heads, pad, flush=True)
    pages, table, cu, lens, rows = _paged.batch(new, total, pad=pad, extra_columns=1, seed=sum(total) + heads)
    _paged.fill(pages, table, total)
    q, qp = queries(rows, heads, 21)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    check(cuda, q, qp, pages, table, cu, lens, out, lse)


@pytest.mark.parametrize("std", [0.02, 4.0])
def test_flat_and_peaked_softmax(cuda, std):
    pages, table, cu, lens, rows = _paged.batch([3, 40], [600, 900], seed=23)
    _paged.fill(pages, table, [600, 900], std=2.0)
    q, qp = queries(rows, 16, 25, std)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    check(cuda, q, qp, pages, table, cu, lens, out, lse)


def test_scores_that_grow_along_the_cache(cuda):
    """Every block of keys raises the running maximum: the sums so far are rescaled again and again."""
    total = [1500, 1400]
    pages, table, cu, lens, rows = _paged.batch([2, 40], total, seed=27)
    _paged.fill(pages, table, total)
    q, qp = queries(rows, 16, 29)
    codes, scales, rope = paged.views(pages)
    for b, n in enumerate(total):  # a rope part that agrees with every query's, growing with the position
        p = torch.arange(n)
        rope[table[b].long()[p // 64], p % 64] = (p[:, None] / 100.0).to(torch.bfloat16).expand(n, 64)
    qp.fill_(0.5)
    out, lse = run(cuda, q, qp, pages, table, cu, lens, scale=0.2)
    check(cuda, q, qp, pages, table, cu, lens, out, lse, 0.2)


@pytest.mark.parametrize("heads", [16, 128])
def test_tokens_that_see_nothing(cuda, heads):
    """More new tokens than keys: the first ones stand before position 0."""
    pages, table, cu, lens, rows = _paged.batch([6, 3], [6, 3], seed=31)
    _paged.fill(pages, table, [6, 3])
    lens[0], lens[1] = 2, -4
    q, qp = queries(rows, heads, 33)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    check(cuda, q, qp, pages, table, cu, lens, out, lse)
    assert torch.isneginf(lse[:4]).all() and torch.isfinite(lse[4:6]).all() and torch.isneginf(lse[6:]).all()


@pytest.mark.parametrize("new", [1, 40])
def test_pages_outside_the_pool_are_not_seen(cuda, new):
    pages, table, cu, lens, rows = _paged.batch([new, new, new], [300, 200, 80], seed=35)
    _paged.fill(pages, table, [300, 200, 80])
    table[0, 1], table[0, 4], table[1, 0], table[2, 0], table[2, 1] = -1, pages.shape[0], 2 ** 31 - 1, -2 ** 31, -7
    lens[1] = 400  # 200 positions past the table
    q, qp = queries(rows, 16, 37)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    check(cuda, q, qp, pages, table, cu, lens, out, lse)
    assert torch.isneginf(lse[2 * new:]).all()


@pytest.mark.parametrize("new", [1, 4, 60])
def test_bad_pages_among_many(cuda, new):
    """Enough pages that a workgroup takes several, bad ones first, last and between them, also the first pages of a cache."""
    total = [4000, 5000, 3500] if new > 4 else [12000, 9000, 15000]
    pages, table, cu, lens, rows = _paged.batch([new] * 3, total, seed=59)
    _paged.fill(pages, table, total)
    g = torch.Generator().manual_seed(61)
    for b, n in enumerate(total):
        need = -(-n // 64)
        bad = torch.randperm(need, generator=g)[:need // 3]
        table[b, bad] = torch.where(bad % 2 == 0, -1, pages.shape[0]).to(torch.int32)
        table[b, :4] = -1
    table[2, :-(-total[2] // 64) - 1] = -3  # one page is left, the last
    q, qp = queries(rows, 16, 63)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    check(cuda, q, qp, pages, table, cu, lens, out, lse)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("new", [1, 40])
def test_a_cache_longer_than_its_table(cuda, new):
    """Positions past the table's columns hold no key: the tokens see the table's, all of them."""
    pages, table, cu, lens, rows = _paged.batch([new, new], [320, 320], seed=55)
    _paged.fill(pages, table, [320, 320])
    lens[0], lens[1] = 320 + 7, 2 ** 31 - 1
    q, qp = queries(rows, 16, 57)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    check(cuda, q, qp, pages, table, cu, lens, out, lse)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("what", ["codes", "scale", "rope", "infinite"])
def test_a_bad_key_reaches_only_the_tokens_that_see_it(cuda, what):
    """A NaN or an infinity in a key: tokens before it are as without it, tokens from it on are not finite."""
    pages, table, cu, lens, rows = _paged.batch([50], [250], seed=39)
    _paged.fill(pages, table, [250])
    q, qp = queries(rows, 16, 41)
    clean, clean_lse = run(cuda, q, qp, pages, table, cu, lens)
    page, row = int(table[0, 220 // 64]), 220 % 64
    codes, scales, rope = paged.views(pages)
    if what == "codes":
        codes.view(torch.uint8)[page, row, 300] = 0x7f
    elif what == "rope":
        rope[page, row, 3] = math.nan
    else:
        scales[page, row] = math.nan if what == "scale" else math.inf
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    assert torch.equal(out[:20], clean[:20]) and torch.equal(lse[:20], clean_lse[:20])
    assert not torch.isfinite(out[20:]).all(-1).any()


def test_repeats_are_equal_bit_for_bit(cuda):
    pages, table, cu, lens, rows = _paged.batch([1, 30, 1], [5000, 400, 77], seed=43)
    _paged.fill(pages, table, [5000, 400, 77])
    q, qp = queries(rows, 16, 45)
    first = run(cuda, q, qp, pages, table, cu, lens)
    for _ in range(3):
        again = run(cuda, q, qp, pages, table, cu, lens)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_lse_is_optional_and_leading_dims_are_free(cuda):
    pages, table, cu, lens, rows = _paged.batch([4], [90], seed=47)
    _paged.fill(pages, table, [90])
    q, qp = queries(rows, 16, 49)
    out, _ = run(cuda, q, qp, pages, table, cu, lens)
    again = torch.zeros(1, rows, 16, 512, dtype=torch.bfloat16, device=cuda)
    d = _paged.to(cuda, q[None], qp[None], pages, table, cu, lens)
    flash_paged_mla(*d, again, model_arch="deepseek_v3_2")
    assert torch.equal(out, again[0])


def test_no_tokens(cuda):
    pages, table, cu, lens, _ = _paged.batch([0], [5], seed=51)
    q, qp = queries(0, 16, 53)
    out, lse = run(cuda, q, qp, pages, table, cu, lens)
    assert out.numel() == 0 and lse.numel() == 0
